"""rptc_kernels.attn_prompt: a row's result depends on that row alone, and on all that it sees."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


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


def randn(seed, *shape, dtype=F16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def ints(xs):
    return torch.tensor(xs, dtype=torch.int32, device="cuda")


# rows, keys, heads, key heads, hd: the forms for few rows (whole, cut), for calls whose longest walk counts (whole, cut), that fill the device
FORMS = [(30, 600, 2, 1, 128), (30, 2500, 2, 1, 128), (512, 512, 32, 8, 128), (400, 400, 32, 8, 64), (150, 3150, 32, 8, 128), (3400, 3400, 32, 8, 64),
         (2600, 2600, 32, 8, 128)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n,L,heads,kvh,hd", FORMS)
def test_a_row_keeps_its_bits_whatever_the_others_are(rk, n, L, heads, kvh, hd, dtype):
    q, k, v = randn(1, n, heads, hd, dtype=dtype), randn(2, L, kvh, hd, dtype=dtype), randn(3, L, kvh, hd, dtype=dtype)

    def attend(q):
        out, lse = torch.empty_like(q), torch.empty(n, heads, device="cuda")
        rk.attn_prompt(q, k, v, out, q_start=ints([0, n]), k_start=ints([0]), k_len=ints([L]), lse=lse, timed=False)
        return out, lse
    out, lse = attend(q)
    for factor in (25.0, 0.0, float("inf")):
        q2 = q.clone()
        q2[3::8] *= factor                                    # rows whose bound is raised far and often, never, or is no number
        out2, lse2 = attend(q2)
        others = torch.arange(n, device="cuda") % 8 != 3
        assert torch.equal(out[others], out2[others]) and torch.equal(lse[others], lse2[others])


@pytest.mark.parametrize("n,L,heads,kvh,hd", [(7, 16384, 4, 4, 64), (64, 16384, 32, 32, 64), (2048, 16384, 16, 16, 64), (300, 8192, 8, 8, 128)])
def test_many_weights_far_below_the_largest(rk, n, L, heads, kvh, hd):
    """The first key outweighs each other one by 2^26 (as the first token of a trained model's context may) and has a value of 0, the others
    of 1: an output is what those weigh together, m / (2^26 + m) with m of them seen.  The scores are hd (exact) and 0, the scale makes the
    one 26 ln 2 to 26 * 2^-23.  fp16 weights are multiples of 2^-24; with the largest at 2^7 at least the others are 32 of those.  Tolerance: the output's half step, the scores' fp32 roundings
    (3 E of the output, E = 18.1 (hd + 4) 2^-24), fp32 sums of at most 2^14 terms of which a lane adds 2^13 (2^-11)."""
    scale = 26 * math.log(2) / hd
    q = torch.ones(n, heads, hd, dtype=F16, device="cuda")
    k, v = torch.zeros(L, kvh, hd, dtype=F16, device="cuda"), torch.ones(L, kvh, hd, dtype=F16, device="cuda")
    k[0], v[0] = 1, 0
    out, lse = torch.empty_like(q), torch.empty(n, heads, device="cuda")
    rk.attn_prompt(q, k, v, out, q_start=ints([0, n]), k_start=ints([0]), k_len=ints([L]), scale=scale, lse=lse, timed=False)
    rest = (torch.arange(n, device="cuda", dtype=torch.float64) + L - n) * 2.0 ** -26
    want = (rest / (1 + rest))[:, None, None]
    E = 18.1 * (hd + 4) * 2.0 ** -24
    assert bool(((out.double() - want).abs() <= want * (2.0 ** -11 + 3 * E + 2.0 ** -11) + 2.0 ** -25).all()), float(((out.double() - want).abs() / want).max())
    assert bool(((lse.double() - hd * scale - torch.log1p(rest)[:, None]).abs() <= 2 * E + 2.0 ** -21 * 20).all())


@pytest.mark.parametrize("n,L,heads,kvh,hd", FORMS)
def test_rows_whose_scores_are_all_minus_infinity(rk, n, L, heads, kvh, hd):
    # every key a row sees has a product of -infinity with it: no weight at all, as for a row that sees no key; its neighbours as ever
    q, k, v = randn(1, n, heads, hd), randn(2, L, kvh, hd), randn(3, L, kvh, hd)
    k[..., 0] = k[..., 0].abs() + 0.1
    q[..., 0] = 0
    out, lse = torch.empty_like(q), torch.empty(n, heads, device="cuda")
    args = dict(q_start=ints([0, n]), k_start=ints([0]), k_len=ints([L]), timed=False)
    rk.attn_prompt(q, k, v, out, lse=lse, **args)
    q2, out2, lse2 = q.clone(), torch.empty_like(q), torch.empty_like(lse)
    q2[5::8, :, 0] = -math.inf
    rk.attn_prompt(q2, k, v, out2, lse=lse2, **args)
    none = torch.arange(n, device="cuda") % 8 == 5
    assert bool((out2[none] == 0).all()) and bool((lse2[none] == -math.inf).all())
    assert torch.equal(out2[~none], out[~none]) and torch.equal(lse2[~none], lse[~none])


@pytest.mark.parametrize("n,L,heads,kvh,hd", FORMS)
def test_one_query_for_all_heads_or_rows(rk, n, L, heads, kvh, hd):
    # a query that is repeated by a stride of 0 gives the bits of its copies
    k, v = randn(2, L, kvh, hd), randn(3, L, kvh, hd)
    args = dict(q_start=ints([0, n]), k_start=ints([0]), k_len=ints([L]), timed=False)
    for q in (randn(1, n, 1, hd).expand(n, heads, hd), randn(1, 1, heads, hd).expand(n, heads, hd), randn(1, 1, 1, hd).expand(n, heads, hd)):
        out, want = torch.empty(n, heads, hd, dtype=F16, device="cuda"), torch.empty(n, heads, hd, dtype=F16, device="cuda")
        rk.attn_prompt(q, k, v, out, **args)
        rk.attn_prompt(q.contiguous(), k, v, want, **args)
        assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n,L,heads,kvh,hd", FORMS)
def test_scores_of_millions_and_more(rk, n, L, heads, kvh, hd, dtype):
    """Scores of 2^28 to 2^37 whose differences, where there are any, are 2^23 and more: one key takes all weight, or those equal to it share it.
    The output is the mean of their values, rounded: each weight is 1, up to 2 roundings of the sum and the quotient, 2^-22."""
    g = torch.Generator(device="cuda").manual_seed(5)
    level = torch.randperm(L, generator=g, device="cuda") // 3                     # every score three times
    size = 60000.0 if dtype == F16 else 2.0 ** 20
    top = (L + 2) // 3
    k = (16 * (level - top / 2).round())[:, None, None].to(dtype).expand(L, kvh, hd).contiguous()      # (their products with q: exact in fp32)
    level = k[:, 0, 0].double()
    q = torch.full((n, heads, hd), size, dtype=dtype, device="cuda")
    q[1::3] *= -1
    q[2::3] = randn(7, 1, heads, hd, dtype=dtype)[:, :, :1] * 0.001                  # rows of ordinary scores between them
    v = randn(8, L, kvh, hd, dtype=dtype)
    out, lse = torch.empty_like(q), torch.empty(n, heads, device="cuda")
    args = dict(q_start=ints([0, n]), k_start=ints([0]), k_len=ints([L]), timed=False)
    rk.attn_prompt(q, k, v, out, lse=lse, **args)
    vd = v.double().repeat_interleave(heads // kvh, 1)
    u = torch.finfo(dtype).eps / 2
    for i in sorted({0, 1, n // 2 // 3 * 3, n // 2 // 3 * 3 + 1, (n - 1) // 3 * 3, n - 1 - (n - 2) % 3}):
        sign = -1 if i % 3 == 1 else 1
        seen = sign * level[:L - n + 1 + i]
        best = seen == seen.max()
        want = vd[:L - n + 1 + i][best].mean(0)
        assert bool(((out[i].double() - want).abs() <= u * want.abs() + 2.0 ** -20).all()), i
        score = size * float(seen.max()) * hd ** 0.5
        assert bool(((lse[i].double() - score - math.log(int(best.sum()))).abs() <= 2.0 ** -20 * abs(score) + 1e-5).all()), i
    # the rows between have the bits they have among their like
    q2, out2, lse2 = q[2::3].repeat_interleave(3, 0)[:n].contiguous(), torch.empty_like(out), torch.empty_like(lse)
    if q2.size(0) < n:
        q2 = torch.cat([q2, q2[-1:].expand(n - q2.size(0), heads, hd)]).contiguous()
    rk.attn_prompt(q2, k, v, out2, lse=lse2, **args)
    assert torch.equal(out[2::3], out2[2::3]) and torch.equal(lse[2::3], lse2[2::3])
