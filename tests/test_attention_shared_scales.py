"""Attention over shared pages with scales of either sign, zero and next to it, in every kernel that a family's size selects."""
import pytest
import torch

from test_attention_shared import Cache

cuda = pytest.mark.gpu


# 4 heads a member: 16, 24, 48, 96 and 160 rows a family
@cuda
@pytest.mark.parametrize("members", [4, 6, 12, 24, 40])
@pytest.mark.parametrize("scale", [0.0, -0.0, -0.1, -2.0, 1e-30, 1e-45, 0.088])
@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.bfloat16, 96), (torch.float32, 128)])
def test_any_scale(members, scale, dtype, dim):
    """The bound of test_attention_shared, with the size of the scale: float32 sums of dim products, the weights' exp carried over to the values
    twice, sums over keys / 32; bfloat16 rounds weights and results to 8 bits."""
    c = Cache([(19, [1, 40, 7] + [5] * (members - 3)), (0, [70])], 8, 2, dim, 16, dtype, members)
    c.scale = scale
    got, want = c.run().double().cpu(), c.want()
    score = max(float((c.q[i].double().norm(dim=1)).max()) for i in range(len(c.kv_len))) * float(c.k.nan_to_num(0.0).double().norm(dim=3).max()) * abs(scale)
    bound = c.value_size * 2.0 ** -24 * (2 * dim * score + max(c.kv_len) / 32 + 64)
    if dtype == torch.bfloat16:
        bound = bound + c.value_size * 2.0 ** -8 + want.abs() * 2.0 ** -8
    off = (got - want).abs()
    assert torch.isfinite(got).all() and (off <= bound).all(), float(off.max())


@cuda
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sizes_of_zero(dtype):
    """No pages, or tables without a column: nobody has a key, and everybody gets zeros.  No heads, no dimensions, pages of no keys: refused."""
    from pulsar_b200 import ops
    from test_attention_shared import on

    def call(pages=3, hq=8, hkv=2, page=16, d=128, width=2):
        q = torch.ones(4, hq, d, dtype=dtype, device="cuda")
        pool, out = torch.zeros(pages, hkv, page, d, dtype=dtype, device="cuda"), torch.full_like(q, 9.0)
        ops.paged_attention_shared(q, pool, pool, out, torch.zeros(4, width, dtype=torch.int32, device="cuda"), on([0] * 4), on([0] * 4), on([]), on([0]), 0, 0, 0.1)
        return out
    for kw in (dict(), dict(pages=0), dict(width=0), dict(pages=0, width=0)):
        assert not call(**kw).any(), kw
    for kw in (dict(page=0), dict(hq=0), dict(hkv=0), dict(d=0)):
        with pytest.raises(ops.KernelError):
            call(**kw)
