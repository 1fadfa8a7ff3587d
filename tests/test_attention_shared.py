"""Attention of one token per sequence over a cache in which families of sequences share pages, against softmax(q k) v in 64 bits."""
import random

import pytest
import torch

from pulsar_b200 import ops

cuda = pytest.mark.gpu


def on(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Cache:
    """Families of sequences over random pages.  ``families``: (shared pages, [own keys of each member]); one with no shared pages is so many
    lone sequences.  Pages and sequences are in no order; every place that no key holds is ``beyond``."""

    def __init__(self, families, hq, hkv, dim, page, dtype, seed, beyond=float("nan"), scale=None):
        rng = random.Random(seed)
        g = torch.Generator().manual_seed(seed)
        total = sum(n for n, _ in families) + sum(-(-k // page) for _, own in families for k in own) + 3
        free = list(range(total))
        rng.shuffle(free)
        seqs = []
        for f, (n_shared, own) in enumerate(families):
            prefix = [free.pop() for _ in range(n_shared)]
            seqs += [(f if n_shared else -1, prefix + [free.pop() for _ in range(-(-k // page))], n_shared * page, n_shared * page + k) for k in own]
        rng.shuffle(seqs)
        n = len(seqs)
        self.k = torch.full((total, hkv, page, dim), beyond).to(dtype)
        self.v = self.k.clone()
        for _, table, _, length in seqs:
            for i, p in enumerate(table):
                rows = min(page, length - i * page)
                if torch.isnan(self.k[p, 0, 0, 0]) or not torch.isfinite(self.k[p, 0, 0, 0]) or self.k[p, 0, 0, 0] == beyond:
                    self.k[p, :, :rows] = torch.randn(hkv, rows, dim, generator=g).to(dtype)
                    self.v[p, :, :rows] = torch.randn(hkv, rows, dim, generator=g).to(dtype)
        self.q = torch.randn(n, hq, dim, generator=g).to(dtype)
        self.tables, self.kv_len, self.shared = [t for _, t, _, _ in seqs], [x for *_, x in seqs], [x for _, _, x, _ in seqs]
        self.members, self.starts = [], [0]
        for f, (n_shared, _) in enumerate(families):
            if n_shared:
                self.members += [i for i, s in enumerate(seqs) if s[0] == f]
                self.starts.append(len(self.members))
        self.most_members = max([b - a for a, b in zip(self.starts, self.starts[1:])], default=0)
        self.page, self.scale, self.dtype = page, scale or dim ** -0.5, dtype

    def run(self, width=0, **changed):
        width = max([1, width] + [len(t) for t in self.tables])
        table = on([t + [-1] * (width - len(t)) for t in self.tables])
        q = self.q.cuda()
        out = torch.full_like(q, 9.0)
        args = dict(q=q, k_pool=self.k.cuda(), v_pool=self.v.cuda(), out=out, block_table=table, kv_len=on(self.kv_len), shared_len=on(self.shared),
                    members=on(self.members), family_start=on(self.starts), most_members=self.most_members, most_shared=max(self.shared, default=0),
                    scale=self.scale)
        args.update(changed)
        ops.paged_attention_shared(**args)
        return args["out"]

    def want(self):
        n, hq, dim = self.q.shape
        hkv = self.k.shape[1]
        out = torch.zeros(n, hq, dim, dtype=torch.float64)
        self.score_size, self.value_size = 0.0, 0.0
        for i in range(n):
            if self.kv_len[i] == 0:
                continue
            k, v = (torch.cat([p[t].double() for t in self.tables[i]], 1)[:, :self.kv_len[i]].repeat_interleave(hq // hkv, 0) for p in (self.k, self.v))
            s = torch.einsum("hd,hnd->hn", self.q[i].double(), k) * self.scale
            out[i] = torch.einsum("hn,hnd->hd", torch.softmax(s, 1), v)
            self.score_size = max(self.score_size, float((self.q[i].double().norm(dim=1) * k.norm(dim=2).amax(1)).max()) * self.scale)
            self.value_size = max(self.value_size, float(v.abs().max()))
        return out

    def check(self, **changed):
        """A score is a sum of dim products: off by up to dim units of its terms' size; the weights' exp carries that over to the values'
        size (twice: above and below the line), a thread adds up to keys / 32 weights.  bfloat16: weights and result are rounded to 8 bits."""
        got, want = self.run(**changed).double().cpu(), self.want()
        unit = 2.0 ** -24
        bound = self.value_size * unit * (2 * self.q.shape[2] * self.score_size + max(self.kv_len) / 32 + 64)
        if self.dtype == torch.bfloat16:
            bound = bound + self.value_size * 2.0 ** -8 + want.abs() * 2.0 ** -8
        off = (got - want).abs()
        assert torch.isfinite(got).all() and (off <= bound).all(), (float(off.max()), float(torch.as_tensor(bound).max()))
        return got


FAMILIES = {
    "one": [(1, [1])],
    "pair": [(3, [5, 21])],
    "eight": [(40, [1, 2, 3, 17, 33, 64, 65, 130])],
    "several": [(9, [4, 40, 7]), (0, [3, 90]), (17, [16, 16]), (1, [200])],
    "alone": [(0, [1, 17, 300])],
    "own_empty": [(5, [0, 0, 3]), (0, [0, 6])],
    "long": [(150, [20, 900]), (2, [1500])],
    "many": [(12, list(range(1, 41)))],
}


@cuda
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("families", FAMILIES)
@pytest.mark.parametrize("hq,hkv,dim,page", [(8, 2, 128, 16), (8, 8, 64, 8), (12, 4, 96, 4), (40, 8, 128, 16), (32, 1, 64, 32), (2, 1, 256, 16), (6, 3, 16, 5), (48, 2, 128, 64)])
def test_against_the_formula(dtype, families, hq, hkv, dim, page):
    Cache(FAMILIES[families], hq, hkv, dim, page, dtype, len(families) * 100 + hq + dim).check()


@cuda
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("beyond", [float("nan"), float("inf"), -float("inf"), 1e30])
def test_what_lies_behind_the_last_key_is_not_read(dtype, beyond):
    Cache([(3, [1, 5, 14]), (0, [9])], 8, 2, 128, 16, dtype, 4, beyond).check()
    Cache([(3, [1, 5, 14]), (0, [9])], 8, 2, 128, 64, dtype, 5, beyond).check()


@cuda
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_scores(dtype):
    """Scores of hundreds: the running maximum rises late, weights under- but nothing overflows."""
    Cache([(20, [40, 3])], 8, 2, 64, 16, dtype, 6, scale=6.0).check()


@cuda
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_family_gives_what_its_members_give_alone(dtype):
    """The same cache with and without the families named: the cut of the keys differs, so the last bits may."""
    c = Cache(FAMILIES["several"], 8, 2, 128, 16, dtype, 7)
    one = c.check()
    c.shared, c.members, c.starts, c.most_members = [0] * len(c.shared), [], [0], 0
    two = c.check()
    assert (one - two).abs().max() <= (2.0 ** -7 if dtype == torch.bfloat16 else 1e-5)


@cuda
def test_wide_tables_scratch_of_the_caller_and_the_same_bits():
    c = Cache(FAMILIES["eight"], 8, 2, 128, 16, torch.bfloat16, 8)
    need = ops.shared_scratch(8, 1, 8, max(c.shared), 400 * 16, 8, 2, 128, 16, torch.bfloat16)
    partial = torch.full((need,), float("nan"), device="cuda")
    first = c.run(width=400, partial=partial)
    assert torch.equal(first, c.run(width=400, partial=partial)) and torch.equal(first, c.run(width=400))
    c.check(width=400, partial=partial)


@cuda
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("families", ["several", "long", "own_empty"])
def test_the_most_own_keys_are_said(dtype, families):
    c = Cache(FAMILIES[families], 8, 2, 128, 16, dtype, 13)
    c.check(width=300, most_own=max(k - s for k, s in zip(c.kv_len, c.shared)))
    c.check(width=300, most_own=4096)


@cuda
def test_offsets_beyond_32_bits():
    """A pool of 4.6 GB whose last pages are read."""
    pages, hkv, page, dim = 70000, 4, 64, 128
    k = torch.zeros(pages, hkv, page, dim, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    v[pages - 1], v[pages - 2] = 2.0, 4.0
    q = torch.ones(2, 8, dim, dtype=torch.bfloat16, device="cuda")
    out = torch.empty_like(q)
    ops.paged_attention_shared(q, k, v, out, on([[pages - 1, pages - 2], [pages - 1, 5]]), on([128, 65]), on([64, 64]), on([1, 0]), on([0, 2]), 2, 64, 0.1)
    assert torch.allclose(out[0].float(), torch.tensor(3.0, device="cuda")) and torch.allclose(out[1].float(), torch.tensor(128 / 65, device="cuda"), rtol=2 ** -7)


@cuda
def test_another_stream_and_a_captured_graph():
    c = Cache(FAMILIES["several"], 8, 2, 64, 16, torch.bfloat16, 9)
    want = c.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = c.run()
    side.synchronize()
    assert torch.equal(got, want)
    width = max(len(t) for t in c.tables)
    kept = [c.q.cuda(), c.k.cuda(), c.v.cuda(), torch.zeros_like(want), on([t + [-1] * (width - len(t)) for t in c.tables]), on(c.kv_len), on(c.shared),
            on(c.members), on(c.starts), c.most_members, max(c.shared), c.scale]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_attention_shared(*kept)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(kept[3], want)


@cuda
def test_refusals():
    c = Cache(FAMILIES["pair"], 8, 2, 64, 16, torch.bfloat16, 10)
    k = c.k.cuda()
    for changed, said in ((dict(out=c.q.float().cuda()), "one dtype"), (dict(kv_len=on(c.kv_len).long()), "int32"), (dict(kv_len=on([1])), "a length"),
                          (dict(most_members=3), "most_members"), (dict(most_shared=-1), "most_members"), (dict(most_own=-1), "most_own"), (dict(v_pool=k[:, :1].contiguous()), "do not fit"),
                          (dict(out=c.q[:1].cuda()), "do not fit"), (dict(partial=torch.empty(3, device="cuda")), "partial"),
                          (dict(family_start=on([])), "one more"), (dict(k_pool=k.transpose(1, 2)), "contiguous")):
        with pytest.raises(ops.KernelError, match=said):
            c.run(**changed)
    d = Cache(FAMILIES["pair"], 4, 2, 24, 16, torch.bfloat16, 11)
    with pytest.raises(ops.KernelError, match="multiple of 16"):
        d.run()
    h = Cache(FAMILIES["pair"], 4, 2, 32, 16, torch.float16, 12)
    with pytest.raises(ops.KernelError, match="float32 or bfloat16"):
        h.run()
    empty = c.q[:0].cuda()
    c.run(q=empty, out=empty.clone(), block_table=on([[0]])[:0], kv_len=on([]), shared_len=on([]), members=on([]), family_start=on([0]), most_members=0)


def test_no_cpu_path():
    z = torch.zeros(1, 2, 16)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ops.KernelError, match="no CPU path"):
        ops.paged_attention_shared(z, torch.zeros(1, 1, 4, 16), torch.zeros(1, 1, 4, 16), z, i.view(1, 1), i, i, i, i, 0, 0, 1.0)


@cuda
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim,page", [(128, 16), (64, 8), (96, 16)])
def test_families_of_unlike_length(dtype, dim, page):
    """The cut of the shared keys follows the longest family: a short one has fewer parts, and nothing is read of those it lacks."""
    families = [(1200 // page, [3, 70]), (1, [5, 9, 1]), (300 // page, [64]), (0, [17, 400]), (64 // page, [0, 2])]
    c = Cache(families, 8, 2, dim, page, dtype, dim + page)
    need = ops.shared_scratch(len(c.shared), len(c.starts) - 1, c.most_members, max(c.shared), max(len(t) for t in c.tables) * page, 8, 2, dim, page, dtype)
    c.check(partial=torch.full((need,), float("nan"), device="cuda"))


@cuda
@pytest.mark.parametrize("group", [1, 3, 4, 5, 8, 9, 16, 17])
def test_groups_of_every_size_in_float32(group):
    """Items of up to 4, 8 and 16 rows take walks of their own, more rows further items."""
    Cache([(9, [1, 63, 64, 65]), (0, [130, 16])], 2 * group, 2, 48, 16, torch.float32, group).check()
