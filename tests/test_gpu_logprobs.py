"""Token log probabilities, entropy and top alternatives (rptc_kernels.token_logprobs) against 64-bit log-softmax.

Tolerances: d = x - max is exact or rounded once (2^-24 |d|); a term exp(d) is off by the factor 1 + c with
c = 2^-23 (1.45 |d| + 2) (the product with log2 e, the instruction's unit in the last place), and terms beyond d = -100
weigh less than 2^-100; the sums have at most n roundings in a thread and log2(threads) over them: with n = 150 additions a thread
l is off by at most (150 + 24) 2^-24 + max c (weighted): together below 2^-15 for the sizes here.  A log probability is
then off by 2^-24 |d| + 2^-15 + 2^-23 |ln l|; the entropy by 2^-15 (1 + |t| / l) and its roundings."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rk():
    import rptc_kernels
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    assert rptc_kernels.library().rptc_init() == 0
    return rptc_kernels


@pytest.fixture(autouse=True)
def _announce(request):
    print(f"\n[case] {request.node.nodeid}", flush=True)
    yield


def outputs(rows, top):
    f = lambda *s: torch.full(s, 77.0, dtype=torch.float32, device="cuda")
    out = {"logprob": f(rows), "entropy": f(rows)}
    if top:
        out["top_ids"] = torch.full((rows, top), -7, dtype=torch.int64, device="cuda")
        out["top_logprobs"] = f(rows, top)
    return out


def order(x, top):
    """ids of the `top` largest of every row, equal ones by the lowest id, not-a-number as -inf."""
    v = torch.where(torch.isnan(x), torch.full_like(x, float("-inf")), x).double()
    return torch.sort(v, dim=-1, descending=True, stable=True).indices[:, :top]


def check(x, tokens, out, top):
    d = x.double()
    logp = torch.log_softmax(d, dim=-1)
    p = logp.exp()
    ent = -(torch.where(p > 0, p * logp, torch.zeros_like(p))).sum(-1)
    ent = torch.where(torch.isnan(logp).any(-1), torch.full_like(ent, float("nan")), ent)

    def same(got, want, tol):
        got = got.double()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        inf = torch.isinf(want)
        assert torch.equal(got[inf], want[inf])
        fin = torch.isfinite(want)
        assert bool(((got - want).abs()[fin] <= tol[fin]).all()), float((got - want).abs()[fin].max())
    ok = (tokens >= 0) & (tokens < x.size(1))
    want = logp.gather(1, tokens.clamp(0, x.size(1) - 1)[:, None])[:, 0]
    want = torch.where(ok, want, torch.full_like(want, float("nan")))
    same(out["logprob"], want, 2.0 ** -15 + 2.0 ** -22 * want.abs())
    same(out["entropy"], ent, 2.0 ** -15 * (2 + 2 * ent.abs()))
    if top:
        ids = order(x, top)
        assert torch.equal(out["top_ids"], ids)
        want = logp.gather(1, ids)
        same(out["top_logprobs"], want, 2.0 ** -15 + 2.0 ** -22 * want.abs())


def logits(seed, rows, vocab, dtype, scale=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(rows, vocab, generator=g, device="cuda") * scale).to(dtype)
    return x, torch.randint(0, vocab, (rows,), generator=g, device="cuda")


F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.mark.parametrize("rows,vocab,dtype,top", [
    (1, 1, F32, 1), (3, 2, F16, 2), (5, 7, BF16, 7), (2, 63, F32, 20), (4, 64, F16, 64), (2, 1000, BF16, 64),
    (1, 32000, F16, 5), (33, 32000, F32, 0), (7, 32001, F16, 32), (3, 50257, BF16, 20), (2, 128257, BF16, 20), (2, 131072, F32, 1),
])
def test_against_log_softmax_in_64_bits(rk, rows, vocab, dtype, top):
    x, tokens = logits(1, rows, vocab, dtype)
    out = outputs(rows, top)
    assert rk.token_logprobs(x, tokens, **out) > 0
    check(x, tokens, out, top)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("offset", [1, 3, 6])
def test_rows_that_begin_anywhere(rk, dtype, offset):
    # a window of a wider matrix: rows at odd distances, no 16-byte alignment
    rows, vocab = 6, 5001
    wide, tokens = logits(2, rows, vocab + 9, dtype)
    x = wide[:, offset:offset + vocab]
    tokens = tokens.clamp(max=vocab - 1)
    out = outputs(rows, 9)
    rk.token_logprobs(x, tokens, timed=False, **out)
    check(x, tokens, out, 9)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_ties_masks_and_rows_without_a_distribution(rk, dtype):
    vocab, top = 20011, 12
    low = torch.finfo(dtype).min
    x = torch.zeros(13, vocab, dtype=dtype, device="cuda")                # row 0: all equal
    x[1] = low                                                            # all at the type's lowest value
    x[2], x[2, [5, 20010, 77]] = float("-inf"), 1.0                       # nearly everything masked
    x[3], x[3, [5, 20010, 77]] = low, torch.tensor([1.0, 2.0, 1.0], dtype=dtype, device="cuda")
    x[4] = float("-inf")                                                  # nothing left
    x[5, 100] = float("nan")
    x[6, 100] = float("inf")
    x[7, 3000:] = 4.0                                                     # ties by the thousand behind a few
    x[7, 19999] = 5.0
    x[8, ::2] = -0.0                                                      # zeros of both signs are equal
    x[9] = torch.arange(vocab, device="cuda").remainder(50).to(dtype)
    x[10] = torch.linspace(-1e4, 1e4, vocab, device="cuda").to(dtype)     # one token takes all
    x[11] = torch.linspace(50, -50, vocab, device="cuda").to(dtype)
    x[12, :8000] = float("nan")
    x[12, 8000:] = float("-inf")
    tokens = torch.tensor([3, 4, 5, 6, 7, 8, 9, 3000, -1, vocab, 20010, 0, 1], device="cuda")
    out = outputs(13, top)
    rk.token_logprobs(x, tokens, timed=False, **out)
    check(x, tokens, out, top)
    out64 = outputs(13, 64)
    rk.token_logprobs(x, tokens, timed=False, **out64)
    check(x, tokens, out64, 64)


def test_each_output_alone_gives_the_same_bits(rk):
    x, tokens = logits(4, 9, 32000, F16)
    full = outputs(9, 5)
    rk.token_logprobs(x, tokens, timed=False, **full)
    for name in full:
        alone = {name: torch.zeros_like(full[name])}
        rk.token_logprobs(x, tokens if name == "logprob" else None, timed=False, **alone)
        assert torch.equal(alone[name], full[name])


def test_another_stream_and_a_graph(rk):
    x, tokens = logits(5, 40, 32000, F32)
    want = outputs(40, 5)
    rk.token_logprobs(x, tokens, timed=False, **want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    o = outputs(40, 5)
    with torch.cuda.stream(side):
        rk.token_logprobs(x, tokens, timed=False, **o)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(o[n], want[n]) for n in want)
    g, o = torch.cuda.CUDAGraph(), outputs(40, 5)
    with torch.cuda.graph(g):
        rk.token_logprobs(x, tokens, timed=False, **o)
    for step in range(3):
        x.mul_(0.9)
        rk.token_logprobs(x, tokens, timed=False, **want)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o[n], want[n]) for n in want)


def test_rows_past_2_31_logits(rk):
    rows, vocab = 17000, 128257
    x = torch.empty((rows, vocab), dtype=BF16, device="cuda")
    assert x.numel() > 1 << 31
    g = torch.Generator(device="cuda").manual_seed(1)
    part = (torch.randn((5, vocab), generator=g, device="cuda") * 2).bfloat16()
    x.zero_()
    x[:5], x[-5:] = part, part
    lp, ids = torch.empty(rows, device="cuda"), torch.empty((rows, 3), dtype=torch.int64, device="cuda")
    rk.token_logprobs(x, torch.arange(rows, device="cuda") % 5, lp, top_ids=ids, timed=False)
    alone, alone_ids = torch.empty(5, device="cuda"), torch.empty((5, 3), dtype=torch.int64, device="cuda")
    rk.token_logprobs(part, torch.arange(rows - 5, rows, device="cuda") % 5, alone, top_ids=alone_ids, timed=False)
    assert torch.equal(lp[-5:], alone) and torch.equal(ids[-5:], alone_ids) and torch.equal(ids[:5], alone_ids)
    assert torch.equal(ids[5:-5], torch.arange(3, device="cuda").expand(rows - 10, 3))       # all equal: the lowest ids


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_tokens_without_probability_and_far_ones(rk, dtype):
    # a token at -inf, at the type's lowest value below a large one, and beside the largest of a flat row
    low = torch.finfo(dtype).min
    x = torch.zeros((5, 300), dtype=dtype, device="cuda")
    x[0, 7], x[1, 7], x[2] = float("-inf"), low, low
    x[3, 5], x[3, 7] = -low, low                      # their difference is beyond fp32 in the wide types
    x[4, 7] = float("nan")
    lp, en = torch.empty(5, device="cuda"), torch.empty(5, device="cuda")
    rk.token_logprobs(x, torch.full((5,), 7, device="cuda"), lp, en, timed=False)
    want = torch.log_softmax(x.double(), -1)[:, 7]
    assert lp[0] == float("-inf") and bool(torch.isnan(lp[4])) and bool(torch.isnan(en[4]))
    assert abs(float(lp[2]) + math.log(300)) < 1e-6 * math.log(300) and abs(float(en[2]) - math.log(300)) < 1e-6 * math.log(300)
    assert abs(float(en[0]) - math.log(299)) < 1e-6 * math.log(299)
    for i in (1, 3):
        # what rounds to fp32's range (-FLT_MAX - ln 299 does: half a step there is 1e31) is a number, what does not is -inf
        w = float(want[i].float())
        assert float(lp[i]) == w if math.isinf(w) else abs(float(lp[i]) / w - 1) < 1e-6
    assert float(en[3]) == 0.0
