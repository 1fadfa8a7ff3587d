"""Log probabilities, ranks, entropies and likeliest tokens of rows of logits, against the formulas in 64 bits."""
import math

import pytest
import torch

from pulsar_b200 import ops

cuda = pytest.mark.gpu


def run(logits, tokens, top=0, rank=True):
    rows = logits.shape[0]
    made = dict(logprob=torch.full((rows,), 7.0, device="cuda"), entropy=torch.full((rows,), 7.0, device="cuda"),
                rank=torch.full((rows,), 7, dtype=torch.int32, device="cuda") if rank else None,
                top_ids=torch.full((rows, top), 7, dtype=torch.int32, device="cuda") if top else None,
                top_logprob=torch.full((rows, top), 7.0, device="cuda") if top else None)
    ops.token_scores(logits, tokens, **made)
    return made


def plain(logits, tokens, top):
    """The definitions in float64, on the host."""
    x = logits.double().cpu()
    t = tokens.long().cpu()
    known = (t >= 0) & (t < x.shape[1])
    t0 = torch.where(known, t, torch.zeros_like(t))
    log_p = torch.log_softmax(x, 1)
    given = x.gather(1, t0.view(-1, 1))
    place = torch.arange(x.shape[1])
    rank = ((x > given) | ((x == given) & (place < t0.view(-1, 1)))).sum(1)
    p = log_p.exp()
    entropy = -torch.where(p > 0, p * log_p, torch.where(torch.isnan(p), p, torch.zeros_like(p))).sum(1)
    order = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    # a stable descending sort keeps equal logits in index order; NaN behind -inf
    ids = torch.argsort(order, dim=1, descending=True, stable=True)
    behind = torch.isnan(x).gather(1, ids)
    ids = ids.gather(1, torch.argsort(behind.int(), dim=1, stable=True))[:, :top]
    log_p = torch.where(log_p < torch.finfo(torch.float32).min, -math.inf, log_p)      # results are float32
    logprob = torch.where(known, log_p.gather(1, t0.view(-1, 1)).squeeze(1), torch.full((len(t),), math.nan, dtype=torch.float64))
    return dict(logprob=logprob, entropy=entropy, rank=torch.where(known, rank, torch.full_like(rank, -1)), top_ids=ids, top_logprob=log_p.gather(1, ids))


def near(got, want, vocab):
    """Every exp and every sum of positive terms is right to about 2^-24 of itself: a thread adds up to vocab / 256 of them, the
    threads' sums go through a dozen more; the two differences and the logarithm add a few units of the result's own size."""
    got, want = got.double().cpu(), want
    both = torch.isnan(want)
    assert torch.equal(torch.isnan(got), both)
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    fine = ~both & ~inf
    bound = 2.0 ** -24 * (vocab / 256 + 64) * (1.0 + want[fine].abs())
    assert (got[fine] - want[fine]).abs().le(bound).all(), (got[fine] - want[fine]).abs().max()


def check(logits, tokens, top, rank=True):
    got, want = run(logits, tokens, top, rank), plain(logits, tokens, top)
    near(got["logprob"], want["logprob"], logits.shape[1])
    near(got["entropy"], want["entropy"], logits.shape[1])
    if rank:
        assert torch.equal(got["rank"].long().cpu(), want["rank"])
    if top:
        assert torch.equal(got["top_ids"].long().cpu(), want["top_ids"])
        near(got["top_logprob"], want["top_logprob"], logits.shape[1])
    return got


def logits_of(rows, vocab, dtype, seed, std=2.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, vocab, generator=g) * std).to(dtype).cuda(), torch.randint(0, vocab, (rows,), generator=g).to(torch.int32).cuda()


DTYPES = [torch.float32, torch.bfloat16]


@cuda
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("top", [0, 1, 5, 32])
@pytest.mark.parametrize("rows,vocab", [(1, 33), (1, 151936), (2, 4099), (3, 257), (7, 1000), (19, 32003), (64, 8192), (200, 511), (700, 40)])
def test_against_the_formulas(dtype, top, rows, vocab):
    logits, tokens = logits_of(rows, vocab, dtype, rows * 1000 + vocab)
    check(logits, tokens, top)


@cuda
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab,top", [(1, 1), (2, 2), (5, 5), (16, 16), (31, 31), (32, 32), (33, 32)])
def test_vocabularies_of_a_few_tokens(dtype, vocab, top):
    logits, tokens = logits_of(9, vocab, dtype, vocab)
    check(logits, tokens, top)


@cuda
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 9001), (40, 3001), (700, 130)])
def test_ties_go_to_the_lower_index(dtype, rows, vocab):
    g = torch.Generator().manual_seed(vocab)
    logits = torch.randint(-2, 3, (rows, vocab), generator=g).to(dtype).cuda()
    logits[0] = 0.0                                     # all equal
    if rows > 1:
        logits[1] = torch.where(torch.arange(vocab, device="cuda") % 2 == 0, 0.0, -0.0).to(dtype)       # zeros of either sign are equal
    tokens = torch.randint(0, vocab, (rows,), generator=g).to(torch.int32).cuda()
    check(logits, tokens, 32)


@cuda
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fill", [-math.inf, "lowest", -1e30])
@pytest.mark.parametrize("left", [0, 1, 3, 50])
def test_masked_rows(dtype, fill, left):
    """Rows in which only a few tokens are left, or none: masked with -inf, with the type's lowest number, with a large one."""
    vocab = 5003
    logits, tokens = logits_of(6, vocab, dtype, left)
    keep = torch.zeros(6, vocab, dtype=torch.bool)
    for r in range(6):
        keep[r, torch.randperm(vocab, generator=torch.Generator().manual_seed(r))[:left]] = True
        if left and r % 2:
            tokens[r] = int(keep[r].nonzero()[0])
    logits = torch.where(keep.cuda(), logits, torch.tensor(torch.finfo(dtype).min if fill == "lowest" else fill, dtype=dtype, device="cuda"))
    check(logits, tokens, 8)


@cuda
@pytest.mark.parametrize("dtype", DTYPES)
def test_values_far_apart_and_the_first_or_last_as_the_largest(dtype):
    vocab = 2051
    logits, tokens = logits_of(8, vocab, dtype, 3)
    logits[0, 0], logits[1, -1], logits[2, 1000] = 80.0, 80.0, 3e38
    logits[3] = torch.linspace(-300, 300, vocab).to(dtype).cuda()
    logits[4] = torch.linspace(300, -300, vocab).to(dtype).cuda()
    logits[5] = -3e38
    logits[6] = 3e38
    check(logits, tokens, 20)


@cuda
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("rows,vocab", [(3, 777), (1, 50001), (300, 100)])
def test_not_a_number_and_infinity(dtype, bad, rows, vocab):
    logits, tokens = logits_of(rows, vocab, dtype, 5)
    logits[0, vocab // 2] = bad
    if rows > 1:
        logits[1] = -math.inf
        logits[1, 3] = bad
        logits[2, int(tokens[2])] = bad
    got, want = run(logits, tokens, 8), plain(logits, tokens, 8)
    for name in ("logprob", "entropy"):
        assert torch.equal(torch.isnan(got[name].cpu()), torch.isnan(want[name]))
    assert torch.equal(got["rank"].long().cpu(), want["rank"]) and torch.equal(got["top_ids"].long().cpu(), want["top_ids"])


@cuda
@pytest.mark.parametrize("dtype", DTYPES)
def test_tokens_outside_the_vocabulary(dtype):
    logits, tokens = logits_of(5, 1234, dtype, 6)
    tokens[1], tokens[2], tokens[4] = -1, 1234, -2 ** 31
    got = check(logits, tokens, 4)
    assert got["rank"].tolist()[1] == got["rank"].tolist()[2] == -1


@cuda
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset", [0, 1, 3])
@pytest.mark.parametrize("stride", [1003, 1024, 2001])
@pytest.mark.parametrize("rows", [1, 5, 333])
def test_rows_at_any_distance_and_address(dtype, offset, stride, rows):
    g = torch.Generator().manual_seed(stride)
    base = (torch.randn(rows * stride + offset + 8, generator=g) * 3).to(dtype).cuda()
    logits = torch.as_strided(base, (rows, 1003), (stride, 1), offset)
    tokens = torch.randint(0, 1003, (rows,), generator=g).to(torch.int32).cuda()
    check(logits, tokens, 6)


@cuda
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("top", [1e3, 5e4, 3e6, 1e20, 3e38, -2e38])
def test_maxima_of_any_size_with_numbers_just_below(dtype, top):
    """The step below a large maximum is a whole number or more: nothing below it weighs anything, and -inf beside the lowest numbers."""
    vocab = 3003
    logits = torch.full((4, vocab), -math.inf, dtype=dtype)
    high = torch.tensor(top, dtype=dtype)
    below = torch.nextafter(high.float(), torch.tensor(-math.inf)).to(dtype) if dtype == torch.float32 else (high.view(torch.int16) + (1 if top < 0 else -1)).view(dtype)
    logits[0, ::3] = below
    logits[0, 1500] = high
    logits[1, ::2] = high
    logits[2, 5::7] = torch.finfo(dtype).min
    logits[3, 5::7] = torch.finfo(dtype).min
    logits[3, 1000] = high
    tokens = torch.tensor([1500, 2000, 5, 1000], dtype=torch.int32)
    check(logits.cuda(), tokens.cuda(), 8)


@cuda
def test_one_row_for_all_and_no_rows():
    logits, _ = logits_of(1, 3001, torch.float32, 8)
    tokens = torch.arange(0, 3001, 60, dtype=torch.int32, device="cuda")
    check(logits.expand(len(tokens), -1), tokens, 3)
    run(logits[:0], tokens[:0], 3)


@cuda
def test_without_ranks_and_alternatives_gives_the_same_numbers():
    logits, tokens = logits_of(33, 7001, torch.float32, 9)
    whole, bare = run(logits, tokens, 20), run(logits, tokens, 0, rank=False)
    assert torch.equal(whole["logprob"], bare["logprob"]) and torch.equal(whole["entropy"], bare["entropy"])


@cuda
def test_the_same_call_gives_the_same_bits():
    logits, tokens = logits_of(5, 151936, torch.float32, 10)
    first = run(logits, tokens, 20)
    for _ in range(3):
        again = run(logits, tokens, 20)
        assert all(torch.equal(first[k], again[k]) for k in first)


@cuda
def test_offsets_beyond_32_bits():
    """20,000 rows of 120,000 bfloat16: the last row starts beyond element 2^31."""
    logits = torch.zeros(20000, 120000, dtype=torch.bfloat16, device="cuda")
    logits[19999, 119999] = 9.0
    logits[17895, 17] = 8.0
    tokens = torch.full((20000,), 119999, dtype=torch.int32, device="cuda")
    got = run(logits, tokens, 2)
    assert got["top_ids"][19999].tolist() == [119999, 0] and got["top_ids"][17895].tolist() == [17, 0]
    assert got["rank"][19999] == 0 and got["rank"][0] == 119999
    assert abs(float(got["logprob"][19999]) - (9.0 - math.log(math.exp(9.0) + 119999))) < 1e-4


@cuda
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 30, 800])
@pytest.mark.parametrize("run_of", [1, 4, 8, 16, 512, 2048, 4096])
def test_large_logits_lie_close_together(dtype, rows, run_of):
    """Runs of large logits, so many apart from each other as a thread's or a block's elements may be: the likeliest lie with few threads."""
    vocab = 60000
    g = torch.Generator().manual_seed(run_of)
    logits = (torch.randn(rows, vocab, generator=g) * 0.5).to(dtype)
    at = torch.arange(vocab)
    logits[:, at % (run_of * 37) < run_of] += 20.0
    logits[::2, at % (run_of * 64) < max(1, run_of // 4)] = 40.0
    tokens = torch.randint(0, vocab, (rows,), generator=g).to(torch.int32).cuda()
    check(logits.cuda(), tokens, 32)


@cuda
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [8192, 16389, 33001, 151937])
def test_the_rank_of_forbidden_tokens(dtype, vocab):
    """The given token is one of many of logit -inf, at the places where a row is cut among blocks and around them."""
    cuts = sorted({min(vocab - 1, max(0, round(vocab * i / 8) + d)) for i in range(9) for d in (-130, -9, -8, -4, -1, 0, 1, 3, 7, 120)})
    logits = torch.full((1, vocab), -math.inf, dtype=dtype)
    logits[0, 5:vocab:1000] = 1.0
    tokens = torch.tensor(cuts, dtype=torch.int32).cuda()
    for some in (tokens[i:i + 1] for i in range(len(cuts))):
        check(logits.cuda(), some, 2)


@cuda
def test_refusals():
    logits, tokens = logits_of(4, 100, torch.float32, 11)
    lp, en = torch.empty(4, device="cuda"), torch.empty(4, device="cuda")
    ids, tlp = torch.empty(4, 3, dtype=torch.int32, device="cuda"), torch.empty(4, 3, device="cuda")
    with pytest.raises(ops.KernelError, match="float32 or bfloat16"):
        ops.token_scores(logits.half(), tokens, lp, en)
    with pytest.raises(ops.KernelError, match="neighbouring"):
        ops.token_scores(logits.t(), tokens, lp, en)
    with pytest.raises(ops.KernelError, match="tokens must be"):
        ops.token_scores(logits, tokens.long(), lp, en)
    with pytest.raises(ops.KernelError, match="entropy must be"):
        ops.token_scores(logits, tokens, lp, en[:3])
    with pytest.raises(ops.KernelError, match="rank must be"):
        ops.token_scores(logits, tokens, lp, en, torch.empty(4, device="cuda"))
    with pytest.raises(ops.KernelError, match="go together"):
        ops.token_scores(logits, tokens, lp, en, None, ids)
    with pytest.raises(ops.KernelError, match="alternatives must be"):
        ops.token_scores(logits, tokens, lp, en, None, ids, tlp[:, :2].contiguous())
    with pytest.raises(ops.KernelError, match="at most 32"):
        ops.token_scores(logits, tokens, lp, en, None, ids.new_empty(4, 33), tlp.new_empty(4, 33))
    with pytest.raises(ops.KernelError, match="at most 32"):
        ops.token_scores(logits[:, :2].contiguous(), tokens, lp, en, None, ids, tlp)
    with pytest.raises(ops.KernelError, match="empty vocabulary"):
        ops.token_scores(logits[:, :0], tokens, lp, en)


def test_no_cpu_path():
    with pytest.raises(ops.KernelError, match="no CPU path"):
        ops.token_scores(torch.zeros(1, 4), torch.zeros(1, dtype=torch.int32), torch.zeros(1), torch.zeros(1))


@cuda
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(297, 65535), (297, 65536), (310, 70001)])
def test_many_long_rows(dtype, rows, vocab):
    """The block's size hangs on the rows, the vocabulary, the type and the alternatives: every row's results, checked on some."""
    logits, tokens = logits_of(rows, vocab, dtype, vocab)
    for top in (0, 20):
        got = run(logits, tokens, top)
        some = torch.tensor([0, 1, 100, 147, 148, 200, rows - 2, rows - 1], device="cuda")
        want = plain(logits[some], tokens[some], top)
        got = {k: v[some] if v is not None else None for k, v in got.items()}
        near(got["logprob"], want["logprob"], vocab)
        near(got["entropy"], want["entropy"], vocab)
        assert torch.equal(got["rank"].long().cpu(), want["rank"])
        if top:
            assert torch.equal(got["top_ids"].long().cpu(), want["top_ids"])
            near(got["top_logprob"], want["top_logprob"], vocab)
