"""Inputs and the 64-bit reference for attention of queries that share rows of the cache, with bounds on what the kernel may be off.

The bounds follow from the arithmetic. The output is sum_j p_j v_j rounded to bf16; the weights p_j reach the tensor cores rounded
to bf16, each by at most 2^-8 of itself (half a step of an 8-bit significand), and are divided by the sum of the unrounded ones:
|error| <= 2^-8 |out| + 2^-8 sum_j p_j |v_j|, where the first term is the final rounding of the perturbed value (hence a factor of
1 + 2^-8). A score is a sum of 576 exact products in fp32: off by at most 576 * 2^-23 * scale * sum_k |q_k k_jk| (tensor cores may
cut instead of rounding), which is also the log-sum-exp's bound, beside its own rounding, and the relative error of a weight twice
over (its own score and the sum's).
"""
import numpy as np
import torch

HEADS, LATENT, ROW = 64, 512, 576


class Case:
    """groups: [(shared, [kv_len of each query])]; one_table: the queries of a group are tokens of one sequence."""

    def __init__(self, groups, one_table=False, block=64, fused=True, gain=1.0, seed=1, extra_blocks=3, heads=HEADS):
        self.block, self.heads, self.scale = block, heads, 1.0 / 24.0
        self.groups, self.one_table = groups, one_table
        blocks_of = lambda n: (n + block - 1) // block  # noqa: E731
        used = sum(blocks_of(s) if one_table else s // block + sum(max(0, blocks_of(n) - s // block) for n in lens) for s, lens in groups)
        self.blocks = used + extra_blocks
        rng = np.random.default_rng(seed)
        order = rng.permutation(self.blocks).tolist()
        columns = max([1] + [blocks_of(max([s] + lens)) for s, lens in groups])
        rows, self.table_index, self.leader, self.shared, self.kv_len = [], [], [], [], []
        for s, lens in groups:
            first = len(self.kv_len)
            common = [order.pop() for _ in range(blocks_of(s) if one_table else s // block)]
            for i, n in enumerate(lens):
                if not one_table or i == 0:
                    row = common + ([] if one_table else [order.pop() for _ in range(max(0, blocks_of(n) - s // block))])
                    rows.append(row + [0] * (columns - len(row)))
                self.table_index.append(len(rows) - 1)
                self.leader.append(first)
                self.shared.append(s if one_table else s // block * block)  # what the table rows have in common: whole blocks
                self.kv_len.append(n)
        self.table = np.array(rows, dtype=np.int32)
        self.batch = len(self.kv_len)
        g = torch.Generator().manual_seed(seed)
        self.pool = torch.randn(self.blocks * block, ROW, generator=g).to(torch.bfloat16)
        self.q = (torch.randn(self.batch, heads, ROW, generator=g) * gain).to(torch.bfloat16)
        self.fused = fused

    def rows_of(self, query, n=None):
        n = self.kv_len[query] if n is None else n
        j = np.arange(n)
        return self.table[self.table_index[query], j // self.block].astype(np.int64) * self.block + j % self.block

    def poison_unused(self, value=float("nan")):
        """Rows that no query attends over hold NaN (also those behind the end inside a sequence's last block)."""
        used = np.zeros(len(self.pool), dtype=bool)
        for b in range(self.batch):
            used[self.rows_of(b)] = True
        self.pool[torch.from_numpy(~used)] = value
        return self

    def want(self):
        """(out, lse, bound of out, bound of lse) in 64 bits."""
        b, h = self.batch, self.heads
        out, a = torch.zeros(b, h, LATENT, dtype=torch.float64), torch.zeros(b, h, LATENT, dtype=torch.float64)
        lse = torch.full((b, h), -float("inf"), dtype=torch.float64)
        score = torch.zeros(b, h, dtype=torch.float64)
        for i in range(b):
            if self.kv_len[i] == 0:
                continue
            k = self.pool[torch.from_numpy(self.rows_of(i))].double()
            q = self.q[i].double()
            s = q @ k.T * self.scale
            lse[i] = torch.logsumexp(s, 1)
            p = torch.exp(s - lse[i][:, None])
            out[i], a[i] = p @ k[:, :LATENT], p @ k[:, :LATENT].abs()
            score[i] = (q.abs() @ k.abs().T).amax(1) * self.scale * 576 * 2.0 ** -23
        bound = 2.0 ** -8 * out.abs() + (1 + 2.0 ** -8) * (2.0 ** -8 + 2 * score)[..., None] * a
        lse_bound = score + torch.where(torch.isfinite(lse), lse.abs(), 0.0) * 2.0 ** -23 + 2.0 ** -21
        return out, lse, bound, lse_bound

    def check(self, out, lse, what=""):
        want, want_lse, bound, lse_bound = self.want()
        off = (out.double().cpu() - want).abs()
        assert not torch.isnan(off).any(), f"{what}: NaN in the output, first at {torch.isnan(off).nonzero()[0].tolist()}"
        worst = (off - bound).amax()
        assert worst <= 0, f"{what}: {(off > bound).sum()} of {off.numel()} outputs beyond the bound by up to {worst:.3e}, first at {(off > bound).nonzero()[0].tolist()}"
        if lse is not None:
            got = lse.double().cpu()
            empty = torch.isinf(want_lse)
            assert (torch.isinf(got) == empty).all() and (got[empty] < 0).all(), f"{what}: log-sum-exp of queries without tokens"
            diff = torch.where(empty, 0.0, got - torch.where(empty, 0.0, want_lse)).abs()
            assert (diff <= lse_bound).all(), f"{what}: log-sum-exp off by {diff.max():.3e}"
