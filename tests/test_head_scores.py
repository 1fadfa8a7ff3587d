"""Log probabilities and entropies straight from hidden rows and the head's weight, against the formulas in 64 bits."""
import math

import pytest
import torch

from pulsar_b200 import ops

cuda = pytest.mark.gpu


def run(h, w, tokens, scale=1.0, cap=None):
    rows = h.shape[0]
    logprob, entropy = torch.full((rows,), 7.0, device="cuda"), torch.full((rows,), 7.0, device="cuda")
    ops.head_scores(h, w, tokens, logprob, entropy, scale, cap)
    return logprob, entropy


def plain(h, w, tokens, scale=1.0, cap=None):
    x = scale * (h.double() @ w.double().t())
    if cap is not None:
        x = cap * torch.tanh(x / cap)
    log_p = torch.log_softmax(x, 1)
    t = tokens.long()
    known = (t >= 0) & (t < w.shape[0])
    got = log_p.gather(1, torch.where(known, t, 0).view(-1, 1)).squeeze(1)
    return torch.where(known, got, math.nan), -torch.special.xlogy(log_p.exp(), log_p.exp()).sum(1)


def check(h, w, tokens, scale=1.0, cap=None):
    """A logit is a sum of K products of at most |h| |w| together, each addition off by a unit of the sum so far (2^-23: the tensor
    cores cut off what the CUDA cores round): over k / 16 or K additions that is K 2^-23 |h| |w| at the very most, and typically its square
    root's share; a sixteenth of it is allowed.  The rest as for logits that are given."""
    got, want = run(h, w, tokens, scale, cap), plain(h, w, tokens, scale, cap)
    k, vocab = h.shape[1], w.shape[0]
    logit = abs(scale) * float(h.double().norm(dim=1).max() * w.double().norm(dim=1).max())
    for a, b in zip(got, want):
        a = a.double()
        assert torch.equal(torch.isnan(a), torch.isnan(b))
        fine = ~torch.isnan(b)
        bound = 2.0 ** -23 * (k / 16 + 16) * logit * (1.0 + b[fine].abs()) / 4 + 2.0 ** -24 * (vocab / 256 + 64) * (1.0 + b[fine].abs())
        assert ((a - b)[fine].abs() <= bound).all(), (float((a - b)[fine].abs().max()), float(bound.min()))


def operands(rows, width, vocab, dtype, seed, std=0.02):
    g = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.randn(rows, width, generator=g, device="cuda").to(dtype)
    w = (torch.randn(vocab, width, generator=g, device="cuda") * std).to(dtype)
    return h, w, torch.randint(0, vocab, (rows,), generator=g, device="cuda").to(torch.int32)


@cuda
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,width,vocab", [(1, 64, 256), (1, 4096, 32003), (2, 8, 1), (3, 72, 17), (17, 1000, 257), (31, 96, 5000), (127, 512, 4099), (128, 128, 40000),
                                              (129, 264, 2500), (200, 640, 151), (256, 1024, 9000), (257, 64, 20011), (700, 200, 3001), (1025, 128, 700)])
def test_against_the_formula(dtype, rows, width, vocab):
    check(*operands(rows, width, vocab, dtype, rows + width + vocab))


@cuda
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scale,cap", [(0.5, None), (1.0, 5.0), (2.5, 30.0), (-1.0, 2.0)])
def test_scale_and_cap(dtype, scale, cap):
    check(*operands(150, 256, 3001, dtype, 5, std=0.1), scale, cap)


@cuda
def test_the_benchmarks_head():
    check(*operands(300, 4096, 151936, torch.bfloat16, 6))


@cuda
@pytest.mark.parametrize("width", [1, 7, 60, 129])
def test_rows_that_are_no_multiple_of_sixteen_bytes(width):
    check(*operands(37, width, 1001, torch.bfloat16, width))


@cuda
def test_addresses_that_are_no_multiple_of_sixteen():
    h, w, tokens = operands(20, 64, 999, torch.bfloat16, 7)
    hb, wb = torch.empty(20 * 64 + 1, dtype=torch.bfloat16, device="cuda"), torch.empty(999 * 64 + 3, dtype=torch.bfloat16, device="cuda")
    h2, w2 = hb[1:].view(20, 64), wb[3:].view(999, 64)
    h2.copy_(h)
    w2.copy_(w)
    check(h2, w2, tokens)


@cuda
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [3, 300])
def test_large_logits_tokens_outside_and_bad_numbers(dtype, rows):
    h, w, tokens = operands(rows, 128, 2003, dtype, 8, std=2.0)       # logits of some 20: a row is nearly certain of one token
    tokens[0], tokens[1] = -1, 2003
    tokens[2] = 2002
    check(h, w, tokens)
    h[1, 5] = math.nan
    got, want = run(h, w, tokens), plain(h, w, tokens)
    for a, b in zip(got, want):
        assert torch.equal(torch.isnan(a), torch.isnan(b))


@cuda
def test_logits_that_fill_more_than_one_slice(monkeypatch):
    h, w, tokens = operands(50, 96, 1003, torch.float32, 9)
    whole = run(h, w, tokens)
    monkeypatch.setattr(ops, "_LOGITS_AT_ONCE", 7 * 1003)
    for a, b in zip(whole, run(h, w, tokens)):
        assert torch.equal(a, b)


@cuda
def test_the_same_bits_on_another_stream():
    h, w, tokens = operands(400, 512, 30001, torch.bfloat16, 10)
    first = run(h, w, tokens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run(h, w, tokens)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    ops.check_wait_words()


@cuda
def test_agrees_with_the_scores_of_the_products_logits():
    h, w, tokens = operands(40, 256, 5003, torch.bfloat16, 11)
    logits = torch.empty(40, 5003, device="cuda")
    ops.linear(h, w, logits)
    lp, en = torch.empty(40, device="cuda"), torch.empty(40, device="cuda")
    ops.token_scores(logits, tokens, lp, en)
    for a, b in zip(run(h, w, tokens), (lp, en)):
        assert (a - b).abs().max() < 2e-5


@cuda
def test_refusals():
    h, w, tokens = operands(4, 64, 100, torch.bfloat16, 12)
    lp, en = torch.empty(4, device="cuda"), torch.empty(4, device="cuda")
    for args, said in (((h, w.float(), tokens, lp, en), "one dtype"), ((h, w[:, :32].contiguous(), tokens, lp, en), "one dtype"),
                       ((h.half(), w.half(), tokens, lp, en), "float32 or bfloat16"), ((h, w, tokens.long(), lp, en), "tokens must be"),
                       ((h, w, tokens, lp[:2], en), "logprob must be"), ((h, w, tokens, lp, en.double()), "entropy must be"),
                       ((h, w, tokens, lp, en, 1.0, 0.0), "cap"), ((h, w, tokens, lp, en, 1.0, -3.0), "cap"), ((h, w[:0], tokens, lp, en), "empty"),
                       ((h.t().contiguous().t(), w, tokens, lp, en), "contiguous")):
        with pytest.raises(ops.KernelError, match=said):
            ops.head_scores(*args)
    ops.head_scores(h[:0], w, tokens[:0], lp[:0], en[:0])


def test_no_cpu_path():
    with pytest.raises(ops.KernelError, match="no CPU path"):
        ops.head_scores(torch.zeros(1, 8), torch.zeros(3, 8), torch.zeros(1, dtype=torch.int32), torch.zeros(1), torch.zeros(1))
