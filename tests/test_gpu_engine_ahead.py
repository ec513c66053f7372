"""Steps of the engine enqueued one behind the other, without waiting for the device in between. The stream stands still while the
host enqueues, so that every upload is still to come when the next step's call is made: each step must reach the device with its own
slots, tables and lengths. What the steps left is compared once, at the end."""
import numpy as np
import pytest
import torch

import b200kv
from shared_cases import HEADS, LATENT, Case

pytestmark = pytest.mark.gpu
LAYERS, BS = 2, 64


class Ahead:
    def __init__(self, **k):
        self.e = b200kv.Engine(**{**dict(layers=LAYERS, max_seqs=6, num_blocks=60, block_size=BS, max_blocks_per_seq=16, max_step_tokens=256, scale=1.0 / 24.0), **k})
        self.rng = torch.Generator().manual_seed(11)
        c, rows = self.e.cache, self.e.config.num_blocks * BS
        self.latent = b200kv.device_tensor(self.e.span_address(c.latent_handle), (LAYERS, rows, 512), torch.bfloat16)
        self.rope = b200kv.device_tensor(self.e.span_address(c.rope_handle), (LAYERS, rows, 64), torch.bfloat16)
        self.gamma = torch.ones(512, dtype=torch.bfloat16, device="cuda")
        self.cos, self.sin = torch.ones(64, dtype=torch.bfloat16, device="cuda"), torch.zeros(64, dtype=torch.bfloat16, device="cuda")
        self.rows = {}      # sequence -> per layer, the producer's inputs of its tokens
        self.done = []      # (layer, sequence, tokens before, tokens of the step, q, out)

    def inputs(self, steps):
        """Everything that the steps [(sequences, tokens each)] read and write, on the device before the first of them."""
        made = []
        for seqs, grow in steps:
            n = sum(grow)
            made.append([(torch.randn(n, 576, generator=self.rng).bfloat16().cuda(), torch.randn(n, HEADS, 576, generator=self.rng).bfloat16().cuda(),
                          torch.full((n, HEADS, LATENT), float("nan"), dtype=torch.bfloat16, device="cuda")) for _ in range(LAYERS)])
        torch.cuda.synchronize()
        return made

    def admit(self, *seqs):
        for s in seqs:
            self.e.admit(s)
            self.rows[s] = [[] for _ in range(LAYERS)]

    def fork(self, src, dst):
        self.e.fork(src, dst)
        self.rows[dst] = [list(of) for of in self.rows[src]]

    def trim(self, s, n):
        self.e.trim(s, n)
        self.rows[s] = [of[:len(of) - n] for of in self.rows[s]]

    def step(self, seqs, grow, made):
        self.e.begin_step(seqs, None if set(grow) == {1} else grow)
        for l, (kv_a, q, out) in enumerate(made):
            self.e.layer_append(l, kv_a, self.gamma, self.cos, self.sin)
            self.e.layer_attend(l, q, out)
            at = 0
            for s, g in zip(seqs, grow):
                self.done.append((l, s, len(self.rows[s][l]), g, q[at:at + g], out[at:at + g]))
                self.rows[s][l] += [kv_a[at + k] for k in range(g)]
                at += g
        self.e.end_step()

    def check(self, skip=()):
        """skip: sequences whose earlier tokens the cache no longer holds."""
        torch.cuda.synchronize()
        assert self.e.status().tolist()[0] == 0
        held = {}
        for s, of in self.rows.items():
            t = np.arange(len(of[0]))
            rows = torch.from_numpy(self.e.table()[s][t // BS].astype(np.int64) * BS + t % BS).cuda()
            for l in range(LAYERS):
                held[s, l] = torch.cat([self.latent[l, rows], self.rope[l, rows]], 1).cpu()
                want = torch.stack(of[l]).cpu()
                assert torch.equal(held[s, l][:, 512:], want[:, 512:]), f"layer {l} sequence {s}: rope rows"
                x = want[:, :512].double()
                x = x / torch.sqrt((x * x).mean(1, keepdim=True) + 1e-6)
                # (half a step of bf16; the norm in fp32: 511 additions are off by at most 2^-15, their root by half of it)
                assert ((held[s, l][:, :512].double() - x).abs() <= (2.0 ** -8 + 2.0 ** -14) * x.abs()).all(), f"layer {l} sequence {s}: latent rows"
        for l, s, had, g, q, out in self.done:
            if s in skip:
                continue
            case = Case([(had + g, [had + k + 1 for k in range(g)])], one_table=True, extra_blocks=0)
            case.table_index, case.table = [0] * g, np.arange((had + g + 63) // 64, dtype=np.int32)[None]
            case.pool = torch.cat([held[s, l][:had + g], torch.zeros(-(had + g) % 64, 576, dtype=torch.bfloat16)])
            case.q = q.cpu()
            case.check(out, None, f"layer {l} sequence {s} with {had} + {g} tokens")


def stand_still():
    torch.cuda._sleep(100_000_000)   # some 50 ms: far longer than it takes to enqueue a step


def test_chunks_and_steps_enqueued_without_waiting():
    a = Ahead()
    a.admit(0, 1, 2)
    steps = [([0], [200]), ([1, 0], [130, 70]), ([2], [5]), ([0, 2, 1], [90, 3, 64]), ([0, 1, 2], [1, 1, 1]), ([2, 0, 1], [1, 1, 1]), ([1], [100]),
             ([1, 2, 0], [1, 1, 1]), ([0, 1], [2, 1])]
    made = a.inputs(steps)
    for i, (step, of) in enumerate(zip(steps, made)):
        if i % 2 == 0:
            stand_still()
        a.step(*step, of)
    a.check()


def test_forks_and_trims_between_steps_enqueued_without_waiting():
    a = Ahead()
    a.admit(0)
    steps = [([0], [190]), ([0, 1, 2], [3, 4, 1]), ([1, 2, 0], [2, 2, 2]), ([0, 1, 2, 3], [1, 1, 1, 1])]
    made = a.inputs(steps)
    stand_still()
    a.step(*steps[0], made[0])
    a.fork(0, 1)
    a.fork(0, 2)
    a.step(*steps[1], made[1])
    stand_still()
    a.trim(1, 3)
    a.step(*steps[2], made[2])
    a.fork(2, 3)
    a.step(*steps[3], made[3])
    a.check(skip=(1,))


def test_an_abandoned_step_between_two_that_wait_their_turn():
    a = Ahead()
    a.admit(0, 1)
    steps = [([0, 1], [70, 66]), ([1, 0], [2, 130]), ([0, 1], [1, 1])]
    made = a.inputs(steps)
    stand_still()
    for step, of in zip(steps, made):
        a.e.begin_step([1, 0], [9, 17])
        a.e.abort_step()
        a.step(*step, of)
    a.check()


def test_a_step_captured_as_a_whole_between_eager_ones():
    a = Ahead()
    a.admit(0)
    steps = [([0], [100]), ([0], [1]), ([0], [3]), ([0], [1]), ([0], [1])]
    made = a.inputs(steps)
    a.step(*steps[0], made[0])
    a.step(*steps[1], made[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):   # (takes the block of the first step, whose upload left an event)
        a.step(*steps[2], made[2])
    graph.replay()
    torch.cuda.synchronize()        # the graph has read the step
    a.step(*steps[3], made[3])
    a.step(*steps[4], made[4])
    a.check()


def test_a_captured_step_uploads_the_step_begun_last():
    """The graph of a decode step, run again for later steps, whose growth an eager call has planned."""
    a = Ahead()
    a.admit(0, 1)
    steps = [([0, 1], [63, 130]), ([0, 1], [1, 1])]
    made = a.inputs(steps)
    a.step(*steps[0], made[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step(*steps[1], made[1])
    for i in range(4):
        if i > 0:
            a.e.begin_step([0, 1])
            for l, (kv_a, q, out) in enumerate(made[1]):
                for k, s in enumerate((0, 1)):
                    a.rows[s][l].append(kv_a[k])
            a.e.end_step()
        graph.replay()
        torch.cuda.synchronize()
        if i > 0:
            a.done = [(l, s, len(a.rows[s][l]) - 1, g, q, out) for l, s, _, g, q, out in a.done if g == 1]
        a.check()
