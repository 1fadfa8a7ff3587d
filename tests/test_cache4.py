"""Keys and values into a cache of 4 bits and back, against the format's definition in 64 bits."""
import pytest
import torch
from cache4 import Cache4, on, quantised, steps_of, values_of, words_of

from pulsar_b200 import ops

cuda = pytest.mark.gpu
BOTH = [torch.float32, torch.bfloat16]


class Rows:
    """Projection rows, their turns and weights, and an empty cache."""

    def __init__(self, n, hq, hkv, dim, page, dtype, rotary=None, norm=True, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.n, self.hq, self.hkv, self.dim, self.page, self.dtype = n, hq, hkv, dim, page, dtype
        self.rotary = dim if rotary is None else rotary
        self.qkv = (2 * torch.randn(n, (hq + 2 * hkv) * dim, generator=g)).to(dtype)
        angle = 40 * torch.rand(n, self.rotary // 2, generator=g)
        self.cos, self.sin = angle.cos(), angle.sin()
        self.weights = [1 + 0.1 * torch.randn(dim, generator=g) if norm else None for _ in range(2)]
        pages = -(-n // page) + 2
        self.slots = torch.randperm(pages * page, generator=g)[:n].to(torch.int32)
        self.pools = [torch.full((pages, hkv, page, dim // 2), 0xab, dtype=torch.uint8), torch.full((pages, hkv, page, dim // 16), 7.0, dtype=torch.bfloat16)] * 2
        self.eps = 1e-6

    def run(self, **changed):
        pools = [p.clone().cuda() for p in self.pools]
        q = torch.full((self.n, self.hq, self.dim), 9.0, dtype=self.dtype, device="cuda")
        args = dict(qkv=self.qkv.cuda(), q_out=q, k_pool=pools[0], k_steps=pools[1], v_pool=pools[2], v_steps=pools[3], slots=self.slots.cuda(), cos=self.cos.cuda(),
                    sin=self.sin.cuda(), q_weight=None if self.weights[0] is None else self.weights[0].cuda(),
                    k_weight=None if self.weights[1] is None else self.weights[1].cuda(), eps=self.eps, n_heads=self.hq, n_kv_heads=self.hkv, head_dim=self.dim,
                    rotary=self.rotary, page_size=self.page)
        args.update(changed)
        ops.qk_norm_rope_write_4bit(**args)
        return [args[k].cpu() for k in ("q_out", "k_pool", "k_steps", "v_pool", "v_steps")]

    def heads(self, first, count, weight):
        """Normed and turned heads in 64 bits."""
        x = self.qkv.double().view(self.n, -1, self.dim)[:, first:first + count]
        if weight is not None:
            x = x / (x.square().mean(-1, keepdim=True) + self.eps).sqrt() * weight.double()
        half = self.rotary // 2
        c, s = self.cos.double().unsqueeze(1), self.sin.double().unsqueeze(1)
        u, v = x[..., :half], x[..., half:2 * half]
        return torch.cat([u * c - v * s, v * c + u * s, x[..., 2 * half:]], -1)

    def want(self):
        q = self.heads(0, self.hq, self.weights[0])
        pools = [p.clone() for p in self.pools]
        k = self.heads(self.hq, self.hkv, self.weights[1]).to(self.dtype).double()
        v = self.qkv.double().view(self.n, -1, self.dim)[:, self.hq + self.hkv:]
        for j, x in ((0, k), (2, v)):
            codes, step, least = quantised(x)
            for i, slot in enumerate(self.slots.tolist()):
                if 0 <= slot < pools[j].shape[0] * self.page:
                    pools[j][slot // self.page, :, slot % self.page] = words_of(codes[i])
                    pools[j + 1][slot // self.page, :, slot % self.page] = steps_of(step[i], least[i])
        return q, pools

    def check(self):
        """Codes and steps are those of the formula, bit for bit: the kernel finds them in 64 bits.  A query is a product of its element, an
        inverse root of a mean of dim squares, a weight and a cosine, added to another such."""
        got, (q, pools) = self.run(), self.want()
        for a, b in zip(got[1:], pools):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        largest = self.heads(0, self.hq, self.weights[0]).abs().amax(-1, keepdim=True) * 2
        bound = largest * 2.0 ** -24 * (self.dim / 2 + 16) + (q.abs() * 2.0 ** -8 if self.dtype == torch.bfloat16 else 0.0)
        assert ((got[0].double() - q).abs() <= bound).all()


@cuda
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("n,hq,hkv,dim,page,rotary,norm", [
    (1, 32, 8, 128, 16, 128, True), (70, 8, 2, 128, 16, 128, True), (5, 4, 4, 32, 4, 32, True), (9, 3, 1, 64, 1, 32, False), (33, 6, 2, 96, 8, 96, True),
    (17, 4, 2, 160, 5, 64, True), (6, 2, 2, 256, 32, 256, True), (3, 0, 2, 128, 16, 0, False), (4, 5, 5, 224, 3, 2, False), (2, 8, 1, 192, 16, 190, True)])
def test_written_as_the_format_says(dtype, n, hq, hkv, dim, page, rotary, norm):
    Rows(n, hq, hkv, dim, page, dtype, rotary, norm, n + dim).check()


@cuda
@pytest.mark.parametrize("dtype", BOTH)
def test_slots_outside_the_pool_are_not_written(dtype):
    r = Rows(9, 4, 2, 64, 4, dtype, seed=3)
    r.slots[2], r.slots[5], r.slots[7] = -1, r.pools[0].shape[0] * 4, 2 ** 31 - 1
    r.check()


@cuda
@pytest.mark.parametrize("dtype", BOTH)
def test_values_of_every_kind(dtype):
    """Constant groups, zeros, one value far from the others, numbers near either end of the range, halves between two codes."""
    r = Rows(12, 1, 2, 64, 4, dtype, rotary=0, norm=False, seed=4)
    x = r.qkv.view(12, 5, 64)
    x[0] = 0.0
    x[1] = -0.0
    x[2] = 3.25
    x[3] = -1e-30
    x[4, :, 7] = 4096.0
    x[5] = 1000.0 + torch.arange(64) / 64
    x[6] *= 1e37
    x[7] *= 1e-37
    x[8] = (torch.arange(64) % 31) / 2                                  # steps of one: every second value lies halfway
    x[9] = torch.where(torch.arange(64) % 2 == 0, 3.3e38, -3.3e38)
    x[10] = 1e-40 * torch.arange(64)
    x[11] = -7.0 - (torch.arange(64) % 16) / 4
    r.check()


@cuda
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_a_group_with_a_value_that_is_no_number_comes_back_as_nan(dtype, value):
    r = Rows(5, 2, 2, 96, 4, dtype, rotary=0, norm=False, seed=5)
    clean = r.run()
    r.qkv.view(5, 6, 96)[3, 2, 40] = value                              # a key's second group
    r.qkv.view(5, 6, 96)[1, 5, 95] = value                              # a value's third group
    got = r.run()
    k, v = (values_of(got[j], got[j + 1])[r.slots.long() // 4, :, r.slots.long() % 4] for j in (1, 3))
    k0, v0 = (values_of(clean[j], clean[j + 1])[r.slots.long() // 4, :, r.slots.long() % 4] for j in (1, 3))
    for a, b, row, head, group in ((k, k0, 3, 0, 1), (v, v0, 1, 1, 2)):
        hit = torch.zeros_like(a, dtype=torch.bool)
        hit[row, head, 32 * group:32 * group + 32] = True
        assert torch.isnan(a[hit]).all() and torch.equal(a[~hit], b[~hit])


@cuda
def test_halves_between_two_codes_of_every_step():
    """Steps of 8 bits from 2^-126 to 2^124, with values on every code and halfway between every two: float32 holds them, and so does the quotient."""
    n = 257
    r = Rows(n, 1, 2, 64, 4, torch.float32, rotary=0, norm=False, seed=35)
    g = torch.Generator().manual_seed(36)
    step = torch.ldexp(torch.randint(128, 256, (n, 5, 2), generator=g).double(), (torch.arange(n) - 140).clamp(-133, 116).view(n, 1, 1))
    x = (step.unsqueeze(-1) * torch.arange(31).double() / 2).float()                                # 0, s / 2, .. 15 s
    least = torch.where(torch.rand(n, 5, 2, 1, generator=g) < 0.5, 0.0, (-step.unsqueeze(-1) * 7).float())
    x = torch.cat([x, x[..., :1]], -1) + least
    r.qkv = x.flatten(1)
    r.check()


@cuda
def test_float32_values_beyond_bfloat16_are_infinite():
    r = Rows(1, 1, 1, 32, 4, torch.float32, rotary=0, norm=False, seed=6)
    r.qkv[0, 40] = 3.4e38
    got = r.run()
    assert torch.isnan(got[2][r.slots[0] // 4, 0, r.slots[0] % 4]).all()


@cuda
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("lens,hkv,dim,page", [([1], 1, 32, 16), ([40, 0, 17, 3], 2, 128, 16), ([9, 33], 3, 96, 4), ([100, 5], 2, 256, 32), ([7, 8, 1], 1, 160, 1), ([50], 4, 64, 24)])
def test_expanded(dtype, lens, hkv, dim, page):
    """Values are a float32 sum of a least value and a product that float32 holds exactly, rounded once to the pages' dtype."""
    c = Cache4(lens, hkv, dim, page, sum(lens))
    table = c.table(width=4)
    table[0, 0] = [-1, table[0, 0].item(), c.pools[0].shape[0]][len(lens) % 3]                 # a page that is none
    s, width = table.shape
    out = [torch.full((s * width + 2, hkv, page, dim), 5.0, dtype=dtype, device="cuda") for _ in range(2)]
    table_out = torch.full_like(table, 77).cuda()
    ops.expand_pages_4bit(*[p.cuda() for p in c.pools], table.cuda(), on(lens), *out, table_out)
    for j, got in zip((0, 2), out):
        want = torch.full(got.shape, 5.0, dtype=dtype)
        wanted_table = torch.full_like(table, -1)
        for i, n in enumerate(lens):
            for p in range(-(-n // page)):
                if not 0 <= table[i, p] < c.pools[j].shape[0]:
                    continue
                x = values_of(c.pools[j][table[i, p]], c.pools[j + 1][table[i, p]]).float().to(dtype)
                x[:, max(0, n - p * page):] = 0.0
                want[i * width + p] = x
                wanted_table[i, p] = i * width + p
        assert torch.equal(got.cpu(), want)
        assert torch.equal(table_out.cpu(), wanted_table)


@cuda
@pytest.mark.parametrize("dtype", BOTH)
def test_what_was_written_comes_back_within_half_a_step(dtype):
    r = Rows(50, 4, 2, 128, 16, dtype, seed=8)
    pages = r.pools[0].shape[0]
    r.slots = torch.arange(50, dtype=torch.int32)
    _, *pools = [t.cuda() for t in r.run()]
    out = [torch.empty(pages, 2, 16, 128, dtype=torch.float32, device="cuda") for _ in range(2)]
    ops.expand_pages_4bit(*pools, on([list(range(pages))]), on([50]), *out, on([[0] * pages]))
    k = r.heads(4, 2, r.weights[1]).to(dtype).double()
    v = r.qkv.double().view(50, -1, 128)[:, 6:]
    for x, got, steps in ((k, out[0], pools[1]), (v, out[1], pools[3])):
        got = got.cpu().double().transpose(1, 2).reshape(-1, 2, 128)[:50]
        step = steps.cpu().double().transpose(1, 2).reshape(-1, 2, 8)[:50, :, 0::2].repeat_interleave(32, -1)
        assert ((got - x).abs() <= step / 2 + got.abs() * 2.0 ** -24).all()


@cuda
def test_another_stream_and_a_captured_graph():
    r = Rows(6, 4, 2, 64, 4, torch.bfloat16, seed=9)
    want = r.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = r.run()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    pools = [p.clone().cuda() for p in r.pools]
    q = torch.empty(6, 4, 64, dtype=torch.bfloat16, device="cuda")
    kept = [r.qkv.cuda(), q, *pools, r.slots.cuda(), r.cos.cuda(), r.sin.cuda(), *[w.cuda() for w in r.weights]]
    out, table = [torch.zeros(4, 2, 4, 64, device="cuda") for _ in range(2)], on([[0, 1, 2, 3]])
    table_out, lens = torch.zeros_like(table), on([16])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.qk_norm_rope_write_4bit(*kept, r.eps, 4, 2, 64, 64, 4)
        ops.expand_pages_4bit(*pools, table, lens, *out, table_out)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(q.cpu(), want[0]) and all(torch.equal(a.cpu(), b) for a, b in zip(pools, want[1:]))
    assert torch.equal(out[0].cpu(), values_of(want[1], want[2]).float())


@cuda
def test_refusals_of_the_writer():
    r = Rows(4, 4, 2, 64, 4, torch.bfloat16, seed=10)
    z = torch.zeros
    for changed, said in ((dict(k_pool=z(3, 2, 4, 64, device="cuda", dtype=torch.uint8)), "codes are uint8"), (dict(v_steps=z(3, 2, 4, 4, device="cuda")), "steps bfloat16"),
                          (dict(qkv=z(4, 500, device="cuda", dtype=torch.bfloat16)), "rows"), (dict(q_out=z(4, 4, 64, device="cuda")), "one dtype"),
                          (dict(slots=r.slots.cuda().long()), "int32"), (dict(slots=r.slots[:3].cuda()), "slots"), (dict(rotary=63), "even number"), (dict(rotary=66), "even number"),
                          (dict(cos=z(4, 30, device="cuda")), "cosines"), (dict(q_weight=z(64, device="cuda", dtype=torch.bfloat16)), "norm weights"), (dict(head_dim=48), "multiple of 32"),
                          (dict(qkv=r.qkv.cuda().half(), q_out=z(4, 4, 64, device="cuda").half()), "float32 or bfloat16"), (dict(qkv=r.qkv), "no CPU path"),
                          (dict(qkv=z(4 * 512 + 4, device="cuda", dtype=torch.bfloat16)[4:].view(4, 512)), "multiple of 16 bytes"),
                          (dict(k_pool=r.pools[0].cuda().transpose(1, 2)), "contiguous"),
                          (dict(k_pool=r.pools[0][:0].cuda(), k_steps=r.pools[1][:0].cuda(), v_pool=r.pools[0][:0].cuda(), v_steps=r.pools[1][:0].cuda()), "without a page")):
        with pytest.raises(ops.KernelError, match=said):
            r.run(**changed)


@cuda
def test_refusals_of_the_expansion():
    c = Cache4([9, 4], 2, 64, 4, 11)

    def run(**changed):
        out = torch.empty(6, 2, 4, 64, device="cuda")
        pools = [p.cuda() for p in c.pools]
        args = dict(k_pool=pools[0], k_steps=pools[1], v_pool=pools[2], v_steps=pools[3], block_table=c.table().cuda(), kv_len=on(c.lens), k_out=out, v_out=out.clone(),
                    table_out=torch.zeros_like(c.table()).cuda())
        ops.expand_pages_4bit(**{**args, **changed})
    run()
    small = torch.empty(5, 2, 4, 64, device="cuda")
    for changed, said in ((dict(k_out=small, v_out=small.clone()), "as many pages"), (dict(v_out=small), "one dtype and shape"), (dict(kv_len=on([9])), "lengths"),
                          (dict(table_out=on([[1, 2]])), "block tables"), (dict(block_table=c.table().cuda().long()), "block tables"),
                          (dict(k_steps=c.pools[1][:3].cuda()), "steps bfloat16"), (dict(k_out=small.half(), v_out=small.half()), "float32 or bfloat16")):
        with pytest.raises(ops.KernelError, match=said):
            run(**changed)
    table = c.table().cuda()
    with pytest.raises(ops.KernelError, match="lie over"):
        run(block_table=table, table_out=table)
    run(block_table=c.table()[:0].cuda(), kv_len=on([]), table_out=c.table()[:0].cuda())
    table_out = c.table().cuda()
    run(k_pool=c.pools[0][:0].cuda(), k_steps=c.pools[1][:0].cuda(), v_pool=c.pools[2][:0].cuda(), v_steps=c.pools[3][:0].cuda(), table_out=table_out)
    assert (table_out == -1).all()


def test_the_format_by_hand():
    """One group, worked out on paper: 0 .. 31 in steps of 31 / 15 rounded up to 8 bits = 2.078125."""
    codes, step, least = quantised(torch.arange(32, dtype=torch.float64))
    assert step.item() == 2.078125 and least.item() == 0.0
    assert codes[0, :6].tolist() == [0, 0, 1, 1, 2, 2] and codes[0, 31] == 15
    words = words_of(codes)
    assert words[0].item() == 0 and words[1].item() == 0x11          # channels 0, 1 in the first byte, 2, 3 in the second
    assert torch.equal(values_of(words, steps_of(step, least)), codes.flatten(-2) * 2.078125)


def test_no_cpu_path():
    u, b, i = torch.zeros(1, 1, 4, 16, dtype=torch.uint8), torch.zeros(1, 1, 4, 2, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ops.KernelError, match="no CPU path"):
        ops.qk_norm_rope_write_4bit(torch.zeros(1, 96), torch.zeros(1, 1, 32), u, b, u, b, i, torch.zeros(1, 0), torch.zeros(1, 0), None, None, 1e-6, 1, 1, 32, 0, 4)
    with pytest.raises(ops.KernelError, match="no CPU path"):
        ops.expand_pages_4bit(u, b, u, b, i.view(1, 1), i, torch.zeros(1, 1, 4, 32), torch.zeros(1, 1, 4, 32), i.view(1, 1))
    with pytest.raises(ops.KernelError, match="no CPU path"):
        ops.paged_attention_4bit(torch.zeros(1, 1, 32), u, b, u, b, torch.zeros(1, 1, 32), i.view(1, 1), i, 1.0)
