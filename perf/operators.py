"""Pages of the cache that several sequences hold, and the attention that reads them, as cases that can be timed and compared.

Two operators: `copy_blocks` moves pages of a paged latent cache in all of its layers at once (the half-filled last page of a
forked sequence, a compaction), and `mla_decode_shared` is decode attention for queries that share rows of the cache: sequences
forked from one prompt, the draft tokens of a step, a chunk of a prompt. Lengths are a function of the case, values of the seed:
latent rows and queries are N(0, 1) bf16 as everywhere in this repository.
"""
import math
import os
import random
import sys

import torch

own = False

HEADS, LATENT, ROPE, ROW = 64, 512, 64, 576
SCALE = 1.0 / 24.0  # 1 / sqrt(576)
_PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ascend-moe-engine_b200")


def _library():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    import b200kv

    return b200kv


def _copy(name, **over):
    case = {"name": name, "kind": "copy", "moves": 1, "rows_lo": 1, "rows_hi": 64, "block": 64, "layers": 43, "blocks": 32, "fused_rows": False}
    case.update(over)
    return case


def _shared(name, **over):
    """`groups` groups of n_lo..n_hi sequences whose first shared_lo..shared_hi tokens are common, each with own_lo..own_hi
    tokens of its own behind them."""
    case = {"name": name, "kind": "shared", "groups": 1, "n_lo": 2, "n_hi": 2, "shared_lo": 1024, "shared_hi": 1024, "own_lo": 1, "own_hi": 64,
            "block": 64, "fused_rows": True, "gain": 1.0}
    case.update(over)
    return case


def _tokens(name, **over):
    """`seqs` sequences of `history_lo..history_hi` tokens, each with new_lo..new_hi tokens of this step behind them, every one of
    which attends up to itself."""
    case = {"name": name, "kind": "tokens", "seqs": 1, "history_lo": 0, "history_hi": 0, "new_lo": 4, "new_hi": 4, "block": 64, "fused_rows": True,
            "gain": 1.0}
    case.update(over)
    return case


def listed():
    return [
        # One sequence is forked: seventeen rows of its last page, in the model's 43 layers.
        _copy("fork_1x17_43layers", rows_lo=17, rows_hi=17),
        # 32 samples of one prompt are forked at once: half-filled pages of 128 tokens.
        _copy("fork_32_43layers", moves=32, rows_hi=127, block=128, blocks=80),
        # A pool is compacted: 300 whole pages move down.
        _copy("compact_300x128_16layers", moves=300, rows_lo=128, rows_hi=128, block=128, layers=16, blocks=640, fused_rows=True),
        # Two samples of a short prompt.
        _shared("prefix_2x1024"),
        # 32 users behind one system prompt, short conversations of their own.
        _shared("prefix_32x4096", n_lo=32, n_hi=32, shared_lo=4096, shared_hi=4096, own_hi=200),
        # Four prompts with some samples each, odd numbers, pages of 128 tokens in two caches, sharper scores.
        _shared("prefix_4groups_ragged", groups=4, n_lo=3, n_hi=11, shared_lo=700, shared_hi=6000, own_lo=0, own_hi=700, block=128, fused_rows=False,
                gain=3.0),
        # Seven questions to one long document.
        _shared("prefix_7x32768", n_lo=7, n_hi=7, shared_lo=32768, shared_hi=32768, own_lo=20, own_hi=300),
        # A full machine behind one long system prompt.
        _shared("prefix_128x8192", n_lo=128, n_hi=128, shared_lo=8192, shared_hi=8192, own_hi=512),
        # Draft tokens to verify: five a sequence.
        _tokens("drafts_16x5", seqs=16, history_lo=300, history_hi=6000, new_lo=5, new_hi=5),
        # Three short prompts, read in one chunk.
        _tokens("prompts_3x200", seqs=3, new_lo=77, new_hi=200, block=128, fused_rows=False),
        # A chunk of a long prompt.
        _tokens("chunk_1024_at_2000", history_lo=2000, history_hi=2000, new_lo=1024, new_hi=1024),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["copy", "shared", "shared", "tokens", "tokens"])
    block, fused, gain = rng.choice([64, 128, 192]), rng.random() < 0.5, rng.choice([1.0, 2.0, 3.0])
    if kind == "copy":
        moves, layers = _log_int(rng, 1, 300), _log_int(rng, 1, 43)
        while moves * layers * block > 300 * 16 * 128:
            moves = (moves + 1) // 2
        rows_lo = rng.randint(1, block)
        case = _copy("", moves=moves, rows_lo=rows_lo, rows_hi=rng.randint(rows_lo, block), block=block, layers=layers,
                     blocks=2 * moves + rng.randint(0, 40), fused_rows=fused)
    elif kind == "shared":
        groups = _log_int(rng, 1, 8)
        n_hi, shared_hi, own_hi = _log_int(rng, 1, 128), _log_int(rng, 1, 32768), _log_int(rng, 1, 800)
        while groups * n_hi * (shared_hi + own_hi) > 128 * 8192:
            if n_hi > 2 and rng.random() < 0.5:
                n_hi //= 2
            elif shared_hi > 100:
                shared_hi //= 2
            else:
                groups = max(1, groups // 2)
        case = _shared("", groups=groups, n_lo=rng.randint(1, n_hi), n_hi=n_hi, shared_lo=rng.randint(0, shared_hi), shared_hi=shared_hi,
                       own_lo=rng.randint(0, own_hi), own_hi=own_hi, block=block, fused_rows=fused, gain=gain)
    else:
        seqs = _log_int(rng, 1, 32)
        history_hi, new_hi = _log_int(rng, 1, 16000), _log_int(rng, 1, 1000)
        while seqs * new_hi * (history_hi + new_hi) > 1024 * 2500:
            if new_hi > 4:
                new_hi //= 2
            else:
                history_hi //= 2
        case = _tokens("", seqs=seqs, history_lo=rng.randint(0, history_hi), history_hi=history_hi, new_lo=rng.randint(1, new_hi), new_hi=new_hi,
                       block=block, fused_rows=fused, gain=gain)
    del case["name"]
    return case


# ---- what follows from a case alone ----------------------------------------------------------------------------------
def _rng(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _move_plan(case):
    """(source, destination, rows) of every move: sources in the upper half of the pool, destinations in the lower."""
    rng = _rng(case)
    half = case["blocks"] // 2
    sources = rng.sample(range(half, case["blocks"]), case["moves"])
    destinations = rng.sample(range(half), case["moves"])
    return [(s, d, rng.randint(case["rows_lo"], case["rows_hi"])) for s, d in zip(sources, destinations)]


def _layout(case):
    """Groups of queries that share a table row's first blocks: [(shared_len, [kv_len of each query])], and whether the queries of
    a group are the tokens of one sequence (one table row) or sequences of their own (a table row each)."""
    rng = _rng(case)
    groups = []
    if case["kind"] == "shared":
        for _ in range(case["groups"]):
            n = rng.randint(case["n_lo"], case["n_hi"])
            shared = rng.randint(case["shared_lo"], case["shared_hi"]) // case["block"] * case["block"]  # whole pages are shared
            groups.append((shared, [shared + rng.randint(case["own_lo"], case["own_hi"]) for _ in range(n)]))
    else:
        for _ in range(case["seqs"]):
            history, new = rng.randint(case["history_lo"], case["history_hi"]), rng.randint(case["new_lo"], case["new_hi"])
            groups.append((history + new, [history + i + 1 for i in range(new)]))
    return groups


def _cache(rows, layers, fused_rows, generator):
    """The pool's storage: latent [layers, rows, 512] and rope [layers, rows, 64], two arrays or columns of one."""
    if fused_rows:
        both = torch.randn(layers, rows, ROW, device="cuda", dtype=torch.bfloat16, generator=generator)
        return both[..., :LATENT], both[..., LATENT:]
    return (torch.randn(layers, rows, LATENT, device="cuda", dtype=torch.bfloat16, generator=generator),
            torch.randn(layers, rows, ROPE, device="cuda", dtype=torch.bfloat16, generator=generator))


def prepare(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    block = case["block"]
    if case["kind"] == "copy":
        state["latent"], state["rope"] = _cache(case["blocks"] * block, case["layers"], case["fused_rows"], generator)
        state["moves"] = torch.tensor(_move_plan(case), dtype=torch.int32, device="cuda")
        if own:
            b200kv = _library()
            latent, rope = state["latent"], state["rope"]
            state["view"] = b200kv.pool_view(latent[0], rope[0])
            state["strides"] = (latent.stride(0), rope.stride(0))
            state["status"] = b200kv.new_status()
        return state

    # A block table as the pool leaves it: blocks in no order, a few pages that nobody holds between them.
    groups = _layout(case)
    one_table = case["kind"] == "tokens"
    blocks_of = lambda tokens: (tokens + block - 1) // block  # noqa: E731
    used = 0
    for shared, lens in groups:
        used += blocks_of(shared) if one_table else shared // block + sum(blocks_of(n) - shared // block for n in lens)
    order = torch.randperm(used + 5, generator=torch.Generator().manual_seed(seed)).tolist()
    columns = max(1, max((blocks_of(max([shared] + lens)) for shared, lens in groups), default=1))
    table, table_index, leader, shared_len, kv_len = [], [], [], [], []
    for shared, lens in groups:
        first = len(kv_len)
        common = [order.pop() for _ in range(blocks_of(shared) if one_table else shared // block)]
        for i, n in enumerate(lens):
            if not one_table or i == 0:
                row = common + ([] if one_table else [order.pop() for _ in range(blocks_of(n) - shared // block)])
                table.append(row + [0] * (columns - len(row)))
            table_index.append(len(table) - 1)
            leader.append(first)
            shared_len.append(shared)
            kv_len.append(n)
    i32 = lambda values: torch.tensor(values, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = len(kv_len)
    latent, rope = _cache((used + 5) * block, 1, case["fused_rows"], generator)
    state.update(latent=latent[0], rope=rope[0], table=i32(table), table_index=i32(table_index), leader=i32(leader), shared_len=i32(shared_len),
                 kv_len=i32(kv_len), groups=groups, batch=batch)
    state["q"] = torch.randn(batch, HEADS, ROW, device="cuda", dtype=torch.bfloat16, generator=generator) * case["gain"]
    if own:
        b200kv = _library()
        state["view"] = b200kv.pool_view(state["latent"], state["rope"])
        state["out"] = torch.empty(batch, HEADS, LATENT, device="cuda", dtype=torch.bfloat16)
        state["lse"] = torch.empty(batch, HEADS, device="cuda", dtype=torch.float32)
        state["workspace"] = torch.empty(b200kv.decode_shared_workspace_bytes(batch), dtype=torch.uint8, device="cuda")
        state["status"] = b200kv.new_status()
    return state


# ---- the plain forms --------------------------------------------------------------------------------------------------
def _plain_copy(state):
    block = state["case"]["block"]
    moves = state["moves"].long()
    offset = torch.arange(block, device="cuda")
    to = moves[:, 1:2] * block + offset
    source = torch.where(offset < moves[:, 2:3], moves[:, 0:1] * block + offset, to)
    for cache in (state["latent"], state["rope"]):
        cache[:, to.reshape(-1)] = cache[:, source.reshape(-1)]
    return [state["latent"], state["rope"]]


def _rows_of(state, query, first, count):
    """Pool rows of tokens first .. first + count - 1 of one query's sequence."""
    block = state["case"]["block"]
    token = torch.arange(first, first + count, device="cuda")
    return state["table"][state["table_index"][query].long()].long()[token // block] * block + token % block


def _plain_attention(state):
    outs, lses = [], []
    first = 0
    for shared, lens in state["groups"]:
        n = len(lens)
        q = state["q"][first:first + n].float() * SCALE
        kv_len = state["kv_len"][first:first + n]
        rows = _rows_of(state, first, 0, shared)
        latent, rope = state["latent"][rows].float(), state["rope"][rows].float()
        scores = q[..., :LATENT] @ latent.T + q[..., LATENT:] @ rope.T  # [n, heads, shared]
        inside = torch.arange(shared, device="cuda") < kv_len[:, None]
        scores = torch.where(inside[:, None, :], scores, -math.inf)
        width = max(0, max(lens) - shared)
        if width:  # each query's own tokens, padded to the longest
            rows = torch.stack([torch.cat([_rows_of(state, first + i, shared, max(0, lens[i] - shared)),
                                           torch.zeros(width - max(0, lens[i] - shared), dtype=torch.long, device="cuda")]) for i in range(n)])
            own_latent, own_rope = state["latent"][rows].float(), state["rope"][rows].float()  # [n, width, ...]
            own_scores = q[..., :LATENT] @ own_latent.transpose(1, 2) + q[..., LATENT:] @ own_rope.transpose(1, 2)
            inside = torch.arange(shared, shared + width, device="cuda") < kv_len[:, None]
            scores = torch.cat([scores, torch.where(inside[:, None, :], own_scores, -math.inf)], dim=2)
        if scores.shape[2] == 0:
            outs.append(torch.zeros(n, HEADS, LATENT, device="cuda"))
            lses.append(torch.full((n, HEADS), -math.inf, device="cuda"))
            first += n
            continue
        top = scores.amax(dim=2, keepdim=True)
        weight = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
        total = weight.sum(dim=2, keepdim=True)
        out = weight[..., :shared] @ latent
        if width:
            out = out + weight[..., shared:] @ own_latent
        outs.append(out / torch.where(total == 0, 1.0, total))
        lses.append((top + torch.log(total)).squeeze(2))
        first += n
    return [torch.cat(outs).to(torch.bfloat16), torch.cat(lses)]


def run(state):
    if state["case"]["kind"] == "copy":
        if not own:
            return _plain_copy(state)
        latent_stride, rope_stride = state["strides"]
        _library().copy_blocks(state["view"], state["moves"], state["case"]["block"], layers=state["case"]["layers"], latent_layer_stride=latent_stride,
                               rope_layer_stride=rope_stride, status=state["status"])
        return [state["latent"], state["rope"]]
    if not own:
        return _plain_attention(state)
    _library().mla_decode_shared(state["q"], state["view"], state["table"], state["kv_len"], state["case"]["block"], SCALE, state["leader"],
                                 state["shared_len"], table_index=state["table_index"], out=state["out"], lse=state["lse"],
                                 workspace=state["workspace"], status=state["status"])
    return [state["out"], state["lse"]]


def work(case):
    if case["kind"] == "copy":
        rows = sum(n for _, _, n in _move_plan(case)) * case["layers"]
        return {"bytes": 2 * rows * ROW * 2 + 12 * case["moves"], "flops": 0}
    rows = pairs = queries = 0
    for shared, lens in _layout(case):
        longest = max(lens)
        rows += min(shared, longest) + sum(max(0, n - shared) for n in lens)
        pairs += sum(lens)
        queries += len(lens)
    # Every row of the cache that some query attends over, once; queries in, outputs and log-sum-exp out; lengths and groups.
    moved = rows * ROW * 2 + queries * (HEADS * (ROW * 2 + LATENT * 2 + 4) + 16)
    return {"bytes": moved, "flops": 2 * (ROW + LATENT) * HEADS * pairs}


def exact(case, seed):
    """Attention one query at a time, in 64 bits; a copy computes nothing."""
    if case["kind"] == "copy":
        return None
    state = prepare(case, seed)
    block = case["block"]
    lens = [n for _, group in state["groups"] for n in group]
    table = state["table"].tolist()
    index = state["table_index"].tolist()
    out = torch.zeros(len(lens), HEADS, LATENT, dtype=torch.float64, device="cuda")
    lse = torch.full((len(lens), HEADS), -math.inf, dtype=torch.float64, device="cuda")
    keys, of = None, None
    for b, n in enumerate(lens):
        if n == 0:
            continue
        if of != index[b]:  # all rows of this table row's sequence, in order
            pages = torch.tensor(table[index[b]], device="cuda")
            rows = (pages[:, None] * block + torch.arange(block, device="cuda")).reshape(-1)
            keys = torch.cat([state["latent"][rows], state["rope"][rows]], dim=1).double()
            of = index[b]
        s = torch.einsum("hk,jk->hj", state["q"][b].double(), keys[:n]) / 24.0
        lse[b] = torch.logsumexp(s, dim=1)
        out[b] = torch.einsum("hj,jv->hv", torch.exp(s - lse[b][:, None]), keys[:n, :LATENT])
    return [out, lse]
