"""Pages copied within a cache's pools and into other pools."""
import pytest
import torch

from pulsar_b200 import ops

cuda = pytest.mark.gpu


def _pool(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    size = torch.empty((), dtype=dtype).element_size()
    n = 1
    for v in shape:
        n *= v
    raw = torch.randint(0, 256, (n * size,), generator=g, dtype=torch.uint8)
    return raw.view(dtype).view(shape).cuda()


def _same(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def _pairs(seed, pages, n):
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    return order[:n].cuda(), order[n:2 * n].cuda()


@cuda
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.uint8, torch.float64])
@pytest.mark.parametrize("shape", [(1, 2, 1), (3, 9, 2, 4, 16), (2, 7, 5), (36, 5, 8, 16, 128), (1, 12, 3, 7, 33), (2, 6, 1, 1, 40000)])
def test_within_pools(dtype, shape):
    pools = [_pool(shape, dtype, 1), _pool((shape[0] + 1, shape[1] + 3, *shape[2:], 3), dtype, 2)]
    src, dst = _pairs(3, shape[1], shape[1] // 2)
    want = [p.clone() for p in pools]
    for p, w in zip(pools, want):
        w[:, dst.long()] = p[:, src.long()]
    ops.copy_pages(pools, pools, src, dst)
    assert all(_same(a, b) for a, b in zip(pools, want))


@cuda
def test_into_other_pools_more_than_one_launch_and_strided_entries():
    """33 pools (more than a launch takes), the sources' entries further apart than their pages reach, one pool empty."""
    wide = [_pool((4, 11, 2, 8, 24), torch.bfloat16, i) for i in range(33)]
    sources = [w[:, 2:9] for w in wide]                       # pages 2 to 8 of every entry
    into = [torch.zeros((4, 5, 2, 8, 24), dtype=torch.bfloat16, device="cuda") for _ in wide]
    sources.append(torch.empty((0, 7, 3), device="cuda"))
    into.append(torch.empty((0, 5, 3), device="cuda"))
    src, dst = torch.tensor([6, 0, 3], dtype=torch.int32, device="cuda"), torch.tensor([1, 4, 0], dtype=torch.int32, device="cuda")
    ops.copy_pages(sources, into, src, dst)
    for a, b in zip(sources[:33], into):
        want = torch.zeros_like(b)
        want[:, dst.long()] = a[:, src.long()]
        assert _same(b, want)


@cuda
@pytest.mark.parametrize("shift", [1, 2, 4, 8, 16, 32])
def test_addresses_of_any_alignment(shift):
    base = _pool((1 << 14,), torch.uint8, 5)
    pool = base[shift:shift + 3 * 8 * 160].view(3, 8, 160)
    before = base.clone()
    src, dst = _pairs(6, 8, 3)
    want = pool.clone()
    want[:, dst.long()] = pool[:, src.long()]
    ops.copy_pages([pool], [pool], src, dst)
    assert _same(pool, want)
    assert torch.equal(base[:shift], before[:shift]) and torch.equal(base[shift + 3 * 8 * 160:], before[shift + 3 * 8 * 160:])


@cuda
def test_ids_outside_a_pool_are_left_out_and_no_pairs_do_nothing():
    pool, into = _pool((2, 6, 40), torch.float32, 7), _pool((2, 4, 40), torch.float32, 8)
    want = into.clone()
    want[:, 2] = pool[:, 5]
    on = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")      # noqa: E731
    ops.copy_pages([pool], [into], on([5, -1, 6, 0, 1]), on([2, 0, 1, 4, -3]))
    assert _same(into, want)
    ops.copy_pages([pool], [into], on([]), on([]))
    ops.copy_pages([], [], on([1]), on([2]))
    assert _same(into, want)


@cuda
def test_more_pages_than_blocks_and_offsets_beyond_32_bits():
    """One pool of 4.3 GB: the last page's bytes are beyond 32 bits, and its first and last pages change places in two calls."""
    pool = torch.zeros((1, 4200, 1 << 20), dtype=torch.uint8, device="cuda")
    pool[:, 0], pool[:, 4199] = 3, 200
    on = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")      # noqa: E731
    ops.copy_pages([pool], [pool], on([4199, 0]), on([17, 4198]))
    assert (pool[0, 17] == 200).all() and (pool[0, 4198] == 3).all() and not pool[0, 16].any() and not pool[0, 4197].any()


@cuda
def test_another_stream():
    side = torch.cuda.Stream()
    pool = _pool((36, 40, 8, 16, 128), torch.bfloat16, 9)
    src, dst = _pairs(10, 40, 20)
    want = pool.clone()
    want[:, dst.long()] = pool[:, src.long()]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.copy_pages([pool], [pool], src, dst)
    side.synchronize()
    assert _same(pool, want)


@cuda
def test_refusals():
    pool = _pool((2, 6, 40), torch.float32, 11)
    ids = torch.tensor([0], dtype=torch.int32, device="cuda")
    with pytest.raises(ops.KernelError, match="int32"):
        ops.copy_pages([pool], [pool], ids.long(), ids)
    with pytest.raises(ops.KernelError, match="as many"):
        ops.copy_pages([pool], [pool], ids, torch.cat([ids, ids]))
    with pytest.raises(ops.KernelError, match="pools to read"):
        ops.copy_pages([pool], [], ids, ids)
    with pytest.raises(ops.KernelError, match="same pages"):
        ops.copy_pages([pool], [pool.bfloat16()], ids, ids)
    with pytest.raises(ops.KernelError, match="same pages"):
        ops.copy_pages([pool], [pool[:, :, :39].contiguous()], ids, ids)
    with pytest.raises(ops.KernelError, match="one behind the other"):
        ops.copy_pages([pool[:, :, :39]], [pool[:, :, :39]], ids, ids)
    with pytest.raises(ops.KernelError, match=r"\[entries, pages"):
        ops.copy_pages([pool[0, 0]], [pool[0, 0]], ids, ids)


def test_no_cpu_path():
    pool, ids = torch.zeros(1, 4, 8), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ops.KernelError, match="no CPU path"):
        ops.copy_pages([pool], [pool], ids, ids)
