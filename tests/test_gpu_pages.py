"""Pages copied inside the cache (b200kv_copy_blocks) against the moves done one by one, bit for bit."""
import numpy as np
import pytest
import torch

import b200kv
from gpu_util import status_ok

pytestmark = pytest.mark.gpu


def _cache(layers, rows, layout, seed=0):
    """bf16 latent [layers, rows, 512] and rope [layers, rows, 64] in storage of the given layout; all storage is returned for
    comparison, so that a write outside the rows shows."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    bits = lambda *shape: torch.randint(-32768, 32768, shape, dtype=torch.int16, device="cuda", generator=g).view(torch.bfloat16)  # noqa: E731
    if layout == "split":
        latent, rope = bits(layers, rows, 512), bits(layers, rows, 64)
        return (latent, rope), latent, rope
    if layout == "fused":
        both = bits(layers, rows, 576)
        return (both,), both[..., :512], both[..., 512:]
    if layout == "layers_apart":
        both = bits(layers, rows + 1, 576)
        return (both,), both[:, :rows, :512], both[:, :rows, 512:]
    both = bits(layers, rows, 600)  # "padded": neither array's rows lie one behind the other
    return (both,), both[..., :512], both[..., 520:584]


def _apply(latent, rope, moves, block):
    for s, d, n in moves:
        if s >= 0 and d >= 0 and n > 0:
            latent[:, d * block:d * block + n] = latent[:, s * block:s * block + n]
            rope[:, d * block:d * block + n] = rope[:, s * block:s * block + n]


def _run(storage, latent, rope, moves, block, status, stream=None):
    b200kv.copy_blocks(b200kv.pool_view(latent[0], rope[0]), torch.tensor(moves, dtype=torch.int32, device="cuda").view(-1, 3), block, layers=latent.shape[0],
                       latent_layer_stride=latent.stride(0), rope_layer_stride=rope.stride(0), status=status, stream=stream)


@pytest.mark.parametrize("layout", ["split", "fused", "layers_apart", "padded"])
@pytest.mark.parametrize("block,layers,moves", [
    (64, 1, 1), (64, 43, 1), (64, 3, 40), (128, 2, 7), (1, 2, 50), (7, 5, 30), (16, 1, 300), (192, 2, 9)])
def test_copies(layout, block, layers, moves):
    rng = np.random.default_rng(block * 1000 + moves)
    blocks = 2 * moves + 3
    order = rng.permutation(blocks)
    plan = [(int(order[i]), int(order[moves + i]), int(rng.integers(0, block + 1))) for i in range(moves)]
    plan[0] = (plan[0][0], plan[0][1], block)
    storage, latent, rope = _cache(layers, blocks * block, layout)
    copy = [s.clone() for s in storage]
    status = b200kv.new_status()
    _run(storage, latent, rope, plan, block, status)
    status_ok(status)
    got = [s.clone() for s in storage]
    for s, c in zip(storage, copy):
        s.copy_(c)
    _apply(latent, rope, plan, block)
    assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(got, storage))


def test_one_source_for_many():
    storage, latent, rope = _cache(3, 40 * 64, "split")
    want_latent, want_rope = latent.clone(), rope.clone()
    plan = [(5, d, 33) for d in range(40) if d != 5]
    _apply(want_latent, want_rope, plan, 64)
    status = b200kv.new_status()
    _run(storage, latent, rope, plan, 64, status)
    status_ok(status)
    assert torch.equal(latent.view(torch.int16), want_latent.view(torch.int16)) and torch.equal(rope.view(torch.int16), want_rope.view(torch.int16))


def test_padding_and_bad_moves():
    """Padding is skipped in silence, a bad move is recorded; neither writes anything, the others are done."""
    good = [(1, 2, 64), (3, 4, 10)]
    for extra, code in [((-1, 5, 64), 0), ((5, -1, 64), 0), ((5, 5, 64), 0), ((5, 6, 0), 0), ((10, 6, 1), 2), ((6, 10, 1), 2), ((5, 6, 65), 2),
                        ((5, 6, -1), 2), ((2 ** 31 - 1, 6, 1), 2)]:
        storage, latent, rope = _cache(2, 10 * 64, "fused")
        want = storage[0].clone()
        _apply(want[..., :512], want[..., 512:], good, 64)
        status = b200kv.new_status()
        _run(storage, latent, rope, [good[0], extra, good[1]], 64, status)
        torch.cuda.synchronize()
        assert status.tolist()[0] == code, extra
        if code:
            assert status.tolist()[1] == 1
        assert torch.equal(storage[0].view(torch.int16), want.view(torch.int16)), extra


def test_behind_the_kernel_that_wrote_the_source_and_in_a_graph():
    storage, latent, rope = _cache(4, 20 * 64, "split")
    status = b200kv.new_status()
    moves = torch.tensor([[1, 2, 64], [3, 4, 17]], dtype=torch.int32, device="cuda")
    view = b200kv.pool_view(latent[0], rope[0])
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        b200kv.copy_blocks(view, moves, 64, 4, latent.stride(0), rope.stride(0), status)
    side.synchronize()
    with torch.cuda.graph(graph):
        latent.add_(1)
        b200kv.copy_blocks(view, moves, 64, 4, latent.stride(0), rope.stride(0), status)
        latent.mul_(2)
    latent.fill_(0)
    for i in range(3):
        latent[:, 64:128] += i
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(latent[:, 64:128], latent[:, 128:192])
    status_ok(status)


def test_offsets_beyond_32_bits():
    """Rows further than 2^31 elements and 2^32 bytes behind the base."""
    layers, rows = 3, 80 * 1024
    latent = torch.zeros(layers, rows, 8192, dtype=torch.bfloat16, device="cuda")  # 1.3 GB a layer, rows 16 KB apart
    last = rows // 64 - 1
    latent[:, :64, :584] = torch.randn(layers, 64, 584, device="cuda").bfloat16()
    status = b200kv.new_status()
    _run((latent,), latent[..., :512], latent[..., 520:584], [(0, last, 64)], 64, status)
    status_ok(status)
    assert torch.equal(latent[:, last * 64:, :512], latent[:, :64, :512]) and torch.equal(latent[:, last * 64:, 520:584], latent[:, :64, 520:584])
    assert (latent[:, last * 64:, 512:520] == 0).all() and (latent[:, last * 64:, 584:] == 0).all()
