"""Forks and drafts through the engine on the device: a prompt read in chunks that attend, samples forked from it, steps of several
draft tokens a sequence of which some are taken back, a compaction in between. After every step the attention is compared with 64
bits over the rows that the sequence's own history says it has; the histories are kept apart from the cache."""
import numpy as np
import pytest
import torch

import b200kv
from gpu_util import to_dev_bf16
from shared_cases import HEADS, LATENT, Case

pytestmark = pytest.mark.gpu
LAYERS, BS = 2, 64


class Run:
    def __init__(self, num_blocks, max_blocks, max_seqs=10, max_step_tokens=300):
        self.e = b200kv.Engine(layers=LAYERS, max_seqs=max_seqs, num_blocks=num_blocks, block_size=BS, max_blocks_per_seq=max_blocks,
                               max_step_tokens=max_step_tokens, scale=1.0 / 24.0)
        self.rng = torch.Generator().manual_seed(3)
        c, rows = self.e.cache, num_blocks * BS
        self.latent = b200kv.device_tensor(self.e.span_address(c.latent_handle), (LAYERS, rows, 512), torch.bfloat16)
        self.rope = b200kv.device_tensor(self.e.span_address(c.rope_handle), (LAYERS, rows, 64), torch.bfloat16)
        self.gamma = torch.ones(512, dtype=torch.bfloat16, device="cuda")
        self.cos, self.sin = torch.ones(64, dtype=torch.bfloat16, device="cuda"), torch.zeros(64, dtype=torch.bfloat16, device="cuda")
        self.history = {}   # sequence -> per layer, its rows as the device has them

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.rng).to(torch.bfloat16).cuda()

    def step(self, seqs, grow=None, quantise=False, q_row=576):
        grow = [1] * len(seqs) if grow is None else grow
        n = sum(grow)
        self.e.begin_step(seqs, None if set(grow) == {1} else grow)
        for l in range(LAYERS):
            kv_a, q = self.normal(n, 576), self.normal(n, HEADS, q_row)[..., :576]
            out = torch.full((n, HEADS, LATENT), float("nan"), dtype=torch.bfloat16, device="cuda")
            fp8 = torch.zeros(n, HEADS * LATENT, dtype=torch.uint8, device="cuda") if quantise else None
            scales = torch.zeros(n, HEADS * LATENT // 32, dtype=torch.uint8, device="cuda") if quantise else None
            self.e.layer_append(l, kv_a, self.gamma, self.cos, self.sin)
            self.e.layer_attend(l, q, out, fp8, scales)
            torch.cuda.synchronize()
            assert self.e.status().tolist()[0] == 0
            if quantise:
                codes, of = torch.zeros_like(fp8), torch.zeros_like(scales)
                b200kv.mx_quant_e4m3(out.view(n, -1), codes, of)
                assert torch.equal(codes, fp8) and torch.equal(of, scales)
            # The new tokens' rows, as the producer left them, join the histories; everything before comes from the histories.
            table, at = self.e.table(), 0
            for s, g in zip(seqs, grow):
                had = len(self.history[s][l])
                t = np.arange(had, had + g)
                rows = torch.from_numpy(table[s][t // BS].astype(np.int64) * BS + t % BS).cuda()
                new = torch.cat([self.latent[l, rows], self.rope[l, rows]], 1).cpu()
                case = Case([(had + g, [had + k + 1 for k in range(g)])], one_table=True, extra_blocks=0)
                case.table_index, case.table = [0] * g, np.arange((had + g + 63) // 64, dtype=np.int32)[None]
                case.pool = torch.cat([self.history[s][l], new, torch.zeros(-(had + g) % 64, 576, dtype=torch.bfloat16)])
                case.q = q[at:at + g].cpu()
                case.check(out[at:at + g], None, f"layer {l} sequence {s} with {had} + {g} tokens")
                self.history[s][l] = torch.cat([self.history[s][l], new])
                at += g
        self.e.end_step()

    def admit(self, s):
        self.e.admit(s)
        self.history[s] = [torch.zeros(0, 576, dtype=torch.bfloat16) for _ in range(LAYERS)]

    def fork(self, src, dst, n=-1):
        self.e.fork(src, dst, n)
        self.history[dst] = [h.clone() if n < 0 else h[:n].clone() for h in self.history[src]]

    def trim(self, s, n):
        self.e.trim(s, n)
        self.history[s] = [h[:len(h) - n] for h in self.history[s]]

    def release(self, s):
        self.e.release(s)
        del self.history[s]


def test_a_prompt_its_samples_and_their_drafts():
    r = Run(num_blocks=60, max_blocks=12)
    r.admit(0)
    for n in (200, 130):          # the prompt in two chunks, the second attending over both
        r.step([0], [n])
    for s in (1, 2, 3):
        r.fork(0, s)
    r.fork(0, 4, 256)             # whole blocks only
    r.step([0, 1, 2, 3, 4], quantise=True)
    r.step([3, 0, 4], [4, 5, 1], quantise=True)   # drafts
    r.trim(3, 3)
    r.trim(0, 5)
    r.trim(4, 100)                # back into a block that others hold
    r.step([4, 3, 0], [2, 2, 2])
    r.release(1)
    assert r.e.compact(2) <= 2
    r.step([0, 2, 3, 4])
    r.fork(4, 1, 0)               # a sequence without tokens
    r.step([1, 4], [70, 1])
    r.release(2)                  # its own last block stands before others'
    assert r.e.compact() > 0
    r.step([1, 4, 0, 3])
    used = {int(b) for s in r.history for b in r.e.table()[s][:(r.e.seq_len(s) + 63) // 64]}
    assert used == set(range(len(used)))


def test_forks_whose_common_blocks_are_many_attend_together():
    """Enough common tokens that a step of one token each goes through the entry point for shared rows."""
    r = Run(num_blocks=320, max_blocks=200, max_step_tokens=4500)
    r.admit(0)
    r.e.begin_step([0], [4500])   # (written, not attended: 64 bits over 4,500 queries would take minutes)
    for l in range(LAYERS):
        r.e.layer_append(l, r.normal(4500, 576), r.gamma, r.cos, r.sin)
    r.e.end_step()
    torch.cuda.synchronize()
    t = np.arange(4500)
    rows = torch.from_numpy(r.e.table()[0][t // BS].astype(np.int64) * BS + t % BS).cuda()
    r.history[0] = [torch.cat([r.latent[l, rows], r.rope[l, rows]], 1).cpu() for l in range(LAYERS)]
    for s in range(1, 9):
        r.fork(0, s)
    r.admit(9)
    r.step([0, 1, 2, 3, 4, 5, 6, 7, 9, 8], quantise=True)
    r.step([9, 8, 7, 6, 5, 4, 3, 2, 1, 0])
    r.step([0, 1, 2, 3, 4, 5, 6, 7, 8], q_row=578)   # query rows that only the other entry point takes
    r.trim(3, 100)
    r.step([3, 4, 5, 6, 7, 8], [1, 2, 1, 1, 3, 1])
