"""Attention over keys and values held in 4 bits, against softmax(q k) v of the values that they stand for in 64 bits."""
import pytest
import torch
from cache4 import Cache4, attended, bound, on

from pulsar_b200 import ops

cuda = pytest.mark.gpu
BOTH = [torch.float32, torch.bfloat16]


class Case:
    def __init__(self, lens, hq, hkv, dim, page, dtype, seed, q_lens=None, window=None, scale=None, beyond=float("nan")):
        self.cache = Cache4(lens, hkv, dim, page, seed, beyond)
        self.q_lens = [1] * len(lens) if q_lens is None else q_lens
        self.q = torch.randn(sum(self.q_lens), hq, dim, generator=torch.Generator().manual_seed(seed + 1)).to(dtype)
        self.portions, self.window, self.scale, self.dtype = q_lens is not None, window, dim ** -0.5 if scale is None else scale, dtype

    def table(self, **how):
        table = self.cache.table(**how)
        if self.window:                            # pages that every query has passed have gone back to the pool
            for i, (n, count) in enumerate(zip(self.cache.lens, self.q_lens)):
                table[i, :max(0, n - count - self.window + 1) // self.cache.page] = -1
        return table

    def args(self, **changed):
        cu = [0]
        for n in self.q_lens:
            cu.append(cu[-1] + n)
        q = self.q.cuda()
        made = dict(q=q, **dict(zip(("k_pool", "k_steps", "v_pool", "v_steps"), (p.cuda() for p in self.cache.pools))), out=torch.full_like(q, 9.0),
                    block_table=self.table().cuda(), kv_len=on(self.cache.lens), scale=self.scale, window=self.window, cu_q=on(cu) if self.portions else None,
                    q_lens=self.q_lens if self.portions else None)
        made.update(changed)
        return made

    def run(self, **changed):
        args = self.args(**changed)
        ops.paged_attention_4bit(**args)
        return args["out"]

    def check(self, **changed):
        got = self.run(**changed).double().cpu()
        want, score_size, value_size = attended(self.cache, self.q, self.q_lens, self.scale, self.window)
        off, most = (got - want).abs(), bound(want, score_size, value_size, self.dtype, max(self.cache.lens))
        assert torch.isfinite(got).all() and (off <= most).all(), (float(off.max()), float(most.max()))
        return got


SIZES = [(32, 8, 128, 16), (8, 8, 64, 8), (12, 4, 96, 4), (40, 8, 128, 16), (32, 1, 64, 32), (2, 1, 256, 16), (6, 3, 32, 5), (24, 2, 128, 64), (3, 3, 160, 1), (8, 1, 192, 24), (36, 2, 224, 16)]


@cuda
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("lens", [[1], [2, 17, 16, 15], [0, 33, 0], [64, 65, 300, 5], [1000, 130]])
@pytest.mark.parametrize("hq,hkv,dim,page", SIZES)
def test_single_tokens(dtype, lens, hq, hkv, dim, page):
    Case(lens, hq, hkv, dim, page, dtype, sum(lens) + dim).check()


@cuda
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("lens,q_lens", [([5], [5]), ([40, 3, 17], [2, 3, 1]), ([100, 0, 64, 30], [20, 0, 1, 30]), ([300, 131], [70, 131]), ([16, 9], [0, 4])])
@pytest.mark.parametrize("hq,hkv,dim,page", SIZES)
def test_portions(dtype, lens, q_lens, hq, hkv, dim, page):
    Case(lens, hq, hkv, dim, page, dtype, sum(lens) + dim, q_lens).check()


@cuda
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("hq,hkv,dim,page", [(32, 8, 128, 16), (8, 1, 64, 8)])
def test_long_portions(dtype, hq, hkv, dim, page):
    Case([700, 260], hq, hkv, dim, page, dtype, 5, [333, 260]).check()
    Case([700, 260, 40], hq, hkv, dim, page, dtype, 6, [333, 1, 40], window=100).check()


@cuda
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("window", [1, 2, 16, 40, 500])
@pytest.mark.parametrize("hq,hkv,dim,page", [(8, 2, 128, 16), (6, 2, 96, 5)])
def test_windows(dtype, window, hq, hkv, dim, page):
    Case([1, 200, 41, 39], hq, hkv, dim, page, dtype, window, window=window).check()
    Case([30, 200, 41], hq, hkv, dim, page, dtype, window, [30, 7, 2], window=window).check()


@cuda
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("beyond", [float("nan"), float("inf"), -float("inf"), 1e30])
@pytest.mark.parametrize("page", [16, 64, 6])
def test_what_lies_behind_the_last_key_is_not_seen(dtype, beyond, page):
    Case([1, 17, 70], 8, 2, 128, page, dtype, 4, beyond=beyond).check()
    Case([12, 17, 70], 8, 2, 128, page, dtype, 4, [12, 3, 33], beyond=beyond).check()


@cuda
@pytest.mark.parametrize("dtype", BOTH)
def test_a_key_that_is_no_number_reaches_those_that_see_it_alone(dtype):
    """The later tokens of a portion see it, the earlier ones do not; a window hides it from the last."""
    c = Case([40], 8, 2, 64, 16, dtype, 7, [12], window=6)
    want = c.run().cpu()
    for pool in (1, 3):
        d = Case([40], 8, 2, 64, 16, dtype, 7, [12], window=6)
        d.cache.pools[pool][d.cache.tables[0][2], 0, 0, 2] = float("nan")          # key 32, kv head 0, its second group
        got = d.run().cpu()
        sees = torch.zeros(12, 8, dtype=torch.bool)
        sees[4:10, :4] = True                                                   # positions 32 .. 37, the query heads of kv head 0
        assert torch.equal(got[~sees], want[~sees])
        hit = got[sees] if pool == 1 else got[sees][:, 32:]
        assert torch.isnan(hit).all()


@cuda
@pytest.mark.parametrize("dtype", BOTH)
def test_pages_that_are_none_are_not_seen(dtype):
    """Ids of -1 and beyond the pool in the middle of a sequence: the others' softmax."""
    c = Case([100], 8, 2, 64, 16, dtype, 8)
    table = c.table()
    table[0, 1], table[0, 4] = -1, c.cache.pools[0].shape[0]
    got = c.run(block_table=table.cuda()).double().cpu()
    k, v = (x.repeat_interleave(4, 0) for x in c.cache.key_values(0))
    keep = torch.tensor([i // 16 not in (1, 4) for i in range(100)])
    score = torch.einsum("hd,hnd->hn", c.q[0].double(), k) * c.scale
    want = torch.einsum("hn,hnd->hd", torch.softmax(score.masked_fill(~keep, -float("inf")), -1), v)
    _, score_size, value_size = attended(c.cache, c.q, [1], c.scale)
    assert ((got[0] - want).abs() <= bound(want, score_size, value_size, dtype, 100)).all()
    assert (c.run(block_table=torch.full_like(table, -1).cuda()) == 0).all()


@cuda
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("scale", [6.0, -0.4, 0.0])
def test_scales_of_every_sign(dtype, scale):
    """Scores of hundreds: the running maximum rises late; a scale of zero gives the mean."""
    Case([200, 40, 3], 8, 2, 64, 16, dtype, 9, scale=scale).check()
    Case([200, 40, 3], 8, 2, 64, 16, dtype, 9, [9, 40, 1], scale=scale).check()


@cuda
@pytest.mark.parametrize("size", [1e-30, 1e-6, 1e6, 1e18])
def test_queries_and_values_of_every_size(size):
    """Queries far from one with keys that make up for it, values far from one."""
    c = Case([130, 20], 8, 2, 128, 16, torch.bfloat16, 10)
    c.q = (c.q.float() * size).to(torch.bfloat16)
    c.cache.pools[1] = (c.cache.pools[1].float() / size).to(torch.bfloat16)
    c.cache.pools[3] = (c.cache.pools[3].float() * size).to(torch.bfloat16)
    c.check()


@cuda
@pytest.mark.parametrize("dtype", BOTH)
def test_query_elements_of_unlike_size(dtype):
    c = Case([90], 8, 2, 128, 16, dtype, 11)
    c.q[:, :, ::7] *= 1000.0
    c.q[:, :, 1::7] *= 2.0 ** -30
    c.q[:, 3] = 0.0
    c.scale = 1e-4
    c.check()


@cuda
@pytest.mark.parametrize("dtype", BOTH)
def test_rows_behind_the_last_sequence_stay(dtype):
    c = Case([30, 9], 8, 2, 64, 16, dtype, 12, [4, 2])
    q = torch.cat([c.q, c.q[:3]]).cuda()
    out = torch.full_like(q, 9.0)
    c.run(q=q, out=out)
    assert (out[6:] == 9.0).all()
    assert torch.equal(out[:6], c.run())


@cuda
def test_wide_tables_and_the_same_bits():
    c = Case([100, 3000, 7], 32, 8, 128, 16, torch.bfloat16, 13)
    first = c.check()
    assert torch.equal(first, c.run().double().cpu())
    c.check(block_table=c.table(width=700).cuda())


# (lengths, tokens or None, query and kv heads, head_dim, page, window, how a call of bfloat16 is dealt out: -n for a cluster of n blocks a head, 0 for even shares)
DEALT = [([30], None, 8, 2, 128, 16, None, -1),
         ([1090, 33, 0], None, 8, 2, 128, 16, None, -8),
         ([2050, 0, 5, 1, 700, 31, 32, 33, 257], None, 36, 9, 64, 3, None, -4),
         ([1500, 40], None, 12, 4, 96, 5, 200, -2),
         ([107 * i + 7 for i in range(18)], None, 16, 8, 128, 16, None, -2),
         ([490, 0, 100, 27] * 10, [5, 0, 3, 5] * 10, 8, 2, 96, 7, None, -1),
         ([1600, 77, 900, 4], [5, 1, 5, 4], 24, 2, 128, 16, None, -4),
         ([14399, 3, 0, 450, 1], None, 8, 1, 128, 16, None, 0),
         ([11000, 2500, 20], [20, 1, 20], 24, 2, 128, 8, None, 0),
         ([11000, 2500, 9000, 20], [20, 1, 3, 20], 24, 2, 128, 8, 5000, 0),
         ([(331 * i) % 1920 for i in range(150)], None, 8, 2, 64, 16, None, 0)]


def dealt_out(case, dtype):
    most = max(case.q_lens)
    return ops.scratch_4bit(len(case.q_lens), most, case.q.shape[1], case.cache.hkv, case.cache.dim, case.table().shape[1], case.cache.page, case.window or 0, dtype)[0]


@cuda
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("lens,q_lens,hq,hkv,dim,page,window,how", DEALT)
def test_every_way_to_deal_a_call_out(dtype, lens, q_lens, hq, hkv, dim, page, window, how):
    c = Case(lens, hq, hkv, dim, page, dtype, len(lens) + dim, q_lens, window=window)
    if dtype == torch.bfloat16:
        assert min(dealt_out(c, dtype), 0) == how
    c.check()
    table = c.cache.table().cuda()
    short = on([n // 3 if q_lens is None else min(n, count + n // 3) for n, count in zip(lens, c.q_lens)])            # the lengths alone say what is read
    few = Case(short.tolist(), hq, hkv, dim, page, dtype, len(lens) + dim, q_lens)
    few.cache.tables, few.cache.pools, few.q, few.window = c.cache.tables, c.cache.pools, c.q, window
    few.check(block_table=table)


def test_portions_of_many_rows_take_expanded_pages():
    for tokens, width, want in ((1, 128, None), (4, 250, None), (64, 250, True), (512, 500, True)):
        assert (ops.expanded_4bit(8, tokens, 32, 8, 128, width, 16, 0, torch.bfloat16) is not None) == bool(want)
        assert ops.expanded_4bit(8, tokens, 32, 8, 128, width, 16, 0, torch.float32) is None
        assert ops.expanded_4bit(8, tokens, 32, 8, 96, width, 6, 0, torch.bfloat16) is None


@cuda
@pytest.mark.parametrize("window", [None, 100])
@pytest.mark.parametrize("room", [1, 3 * 4 * 25 * 2 * 16 * 128])
def test_expanded_pages_of_a_few_sequences_at_a_time(room, window, monkeypatch):
    """Sequences over whose pages too much room would go are taken in runs; rows of none stay."""
    c = Case([400, 130, 0, 390, 64, 100, 40], 8, 2, 128, 16, torch.bfloat16, 31, [300, 130, 0, 260, 0, 100, 33], window=window)
    monkeypatch.setattr(ops, "_expanded_pays_4bit", lambda *a: True)
    want = c.check()
    monkeypatch.setattr(ops, "EXPANDED_ROOM_4BIT", room)
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    got = c.run()
    assert torch.equal(got.double().cpu(), want)
    assert torch.cuda.max_memory_allocated() - before < max(room, 4 * 25 * 2 * 16 * 128) + 8 * c.q.numel() + (4 << 20)


@cuda
@pytest.mark.parametrize("q_lens", [None, [90, 33, 200]])
def test_windows_as_wide_as_all_keys_and_queries_as_outputs(q_lens):
    c = Case([90, 33, 400], 8, 2, 128, 16, torch.bfloat16, 33, q_lens)
    want = c.run()
    for window in (401, (1 << 31) - 1, 1 << 40):
        assert torch.equal(c.run(window=window), want)
    if q_lens is None:                         # a row of q is read before anything is written to it
        q = c.q.cuda()
        assert torch.equal(c.run(q=q, out=q), want)


@cuda
@pytest.mark.parametrize("lens,q_lens,window", [([400, 130], [5, 130], None), ([300, 1, 20], [3, 1, 20], 7), ([64], [64], None), ([1], [1], None)])
@pytest.mark.parametrize("hq,hkv,dim,page", [(32, 8, 128, 16), (8, 1, 64, 8), (4, 4, 128, 64)])
def test_either_way_of_portions(lens, q_lens, window, hq, hkv, dim, page, monkeypatch):
    """Short portions over expanded pages, long ones on codes: whichever way a rule takes, the sums are the formula's."""
    c = Case(lens, hq, hkv, dim, page, torch.bfloat16, 32, q_lens, window=window)
    for pays in (True, False):
        monkeypatch.setattr(ops, "_expanded_pays_4bit", lambda *a: pays)
        c.check()


@cuda
def test_one_and_two_heads_a_block_give_the_same_bits(monkeypatch):
    c = Case([700, 260], 16, 4, 128, 16, torch.bfloat16, 34, [333, 260])
    monkeypatch.setattr(ops, "_expanded_pays_4bit", lambda *a: True)
    got = []
    for one in (True, False):
        monkeypatch.setattr(ops, "_one_head_a_block", lambda *a: one)
        got.append(c.check())
    assert torch.equal(*got)


@cuda
def test_many_sequences_of_unlike_length():
    lens = [(37 * i) % 900 for i in range(150)]
    Case(lens, 8, 2, 64, 16, torch.bfloat16, 14).check()
    Case(lens, 4, 4, 32, 8, torch.float32, 15, [min(n, i % 5) for i, n in enumerate(lens)]).check()


@cuda
def test_offsets_beyond_32_bits():
    """A pool of 4.6 GB of codes whose last pages are read and written."""
    pages, hkv, page, dim = 140000, 8, 64, 128
    codes = torch.zeros(pages, hkv, page, dim // 2, dtype=torch.uint8, device="cuda")
    steps = torch.zeros(pages, hkv, page, dim // 16, dtype=torch.bfloat16, device="cuda")
    last = steps[pages - 2:].view(2, hkv, page, dim // 32, 2)
    last[..., 0] = 1.0
    codes[pages - 1], codes[pages - 2] = 0x22, 0x44
    q = torch.ones(2, 8, dim, dtype=torch.bfloat16, device="cuda")
    out = torch.empty_like(q)
    ops.paged_attention_4bit(q, codes, steps, codes, steps, out, on([[pages - 1, pages - 2], [5, pages - 1]]), on([1, 65]), 0.0)
    assert (out[0] == 2.0).all() and torch.allclose(out[1].float(), torch.tensor(2.0 / 65, device="cuda"), rtol=2.0 ** -7)
    slot = on([(pages - 1) * page + 63])
    qkv = torch.ones(1, (8 + 16) * dim, dtype=torch.bfloat16, device="cuda")
    ops.qk_norm_rope_write_4bit(qkv, q[:1].clone(), codes, steps, codes, steps, slot, torch.zeros(1, 0, device="cuda"), torch.zeros(1, 0, device="cuda"), None, None, 1e-6, 8, 8, dim, 0, page)
    assert (steps[pages - 1, :, 63].view(hkv, -1, 2) == torch.tensor([0.0, 1.0], device="cuda")).all() and (codes[pages - 1, :, 63] == 0).all()
    out_k = torch.empty(1, hkv, page, dim, device="cuda")
    ops.expand_pages_4bit(codes, steps, codes, steps, on([[pages - 1]]), on([64]), out_k, out_k.clone(), on([[0]]))
    assert (out_k[0, :, 63] == 1.0).all() and (out_k[0, :, :63] == 2.0).all()


@cuda
@pytest.mark.parametrize("q_lens", [None, [3, 40, 1], [200, 90, 64]])
def test_another_stream_and_two_captured_graphs(q_lens):
    """Two graphs of the same sizes, replayed one behind the other and again: neither's workspace is the other's."""
    a, b = (Case([300, 90, 64], 8, 2, 128, 16, torch.bfloat16, seed, q_lens) for seed in (16, 17))
    want = [c.run() for c in (a, b)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = a.run()
    side.synchronize()
    assert torch.equal(got, want[0])
    kept, graphs = [c.args() for c in (a, b)], []
    torch.cuda.synchronize()
    for args in kept:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.paged_attention_4bit(**args)
        graphs.append(graph)
    for _ in range(2):
        for args in kept:
            args["out"].zero_()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(args["out"], w) for args, w in zip(kept, want))


@cuda
def test_two_calls_at_once():
    cases = [Case([2000, 900], 8, 2, 128, 16, torch.bfloat16, seed) for seed in (18, 19)]
    args = [c.args() for c in cases]
    want = [c.run() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(20):
        for a, s in zip(args, streams):
            with torch.cuda.stream(s):
                ops.paged_attention_4bit(**a)
    torch.cuda.synchronize()
    assert all(torch.equal(a["out"], w) for a, w in zip(args, want))


@cuda
def test_refusals():
    c = Case([20, 5], 8, 2, 64, 16, torch.bfloat16, 20, [2, 1])
    q = c.q.cuda()
    for changed, said in ((dict(out=q.float()), "one dtype"), (dict(out=q[:1]), "one dtype"), (dict(kv_len=on([20])), "lengths"), (dict(kv_len=on([20, 5]).long()), "lengths"),
                          (dict(cu_q=None), "go together"), (dict(cu_q=None, q_lens=None), "one query token"), (dict(q_lens=[2]), "numbers of tokens"),
                          (dict(q_lens=[3, 1]), "numbers of tokens"), (dict(q_lens=[-1, 1]), "numbers of tokens"), (dict(cu_q=on([0, 3])), "numbers of tokens"),
                          (dict(window=0), "window"), (dict(window=-3), "window"), (dict(v_pool=c.cache.pools[2][:, :1].cuda()), "codes are uint8"),
                          (dict(v_steps=c.cache.pools[3].float().cuda()), "steps bfloat16"), (dict(q=q[:, :7].contiguous(), out=q[:, :7].contiguous()), "cannot be grouped"),
                          (dict(block_table=c.table().cuda().long()), "block table"), (dict(q=q.half(), out=q.half()), "float32 or bfloat16"), (dict(q=q.cpu()), "no CPU path"),
                          (dict(k_pool=c.cache.pools[0].cuda().transpose(1, 2)), "contiguous")):
        with pytest.raises(ops.KernelError, match=said):
            c.run(**changed)
    d = Case([20], 4, 2, 32, 16, torch.bfloat16, 21)
    with pytest.raises(ops.KernelError, match="multiple of 32"):
        d.run(q=torch.zeros(1, 4, 48, dtype=torch.bfloat16, device="cuda"), out=torch.zeros(1, 4, 48, dtype=torch.bfloat16, device="cuda"))
    none = q[:0]
    assert c.run(q=none, out=none.clone(), cu_q=on([0, 0, 0]), q_lens=[0, 0]).numel() == 0
    c.run(q=none, out=none.clone(), block_table=c.table()[:0].cuda(), kv_len=on([]), cu_q=None, q_lens=None)
    assert (c.run(block_table=c.table()[:, :0].contiguous().cuda()) == 0).all()
    empty = [p[:0].cuda() for p in c.cache.pools]
    assert (c.run(k_pool=empty[0], k_steps=empty[1], v_pool=empty[2], v_steps=empty[3]) == 0).all()
