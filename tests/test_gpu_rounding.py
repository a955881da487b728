"""How near the prompt attention, the attention over the 4-bit cache and the token log probabilities come to 64-bit arithmetic in the mean
over many elements, where a bound on each element leaves room for a rounding more.

A result that is exact up to its own rounding is off by what rounding the 64-bit result to its type is off by: that is measured on the
same elements (`own`).  Errors of independent roundings add up as squares: one more rounding of every weight, of a relative size like
the output's own, makes it 1.2 to 1.4 times `own` at the sizes here; the bound between, 1.1, is what two terms a weight have to keep."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


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


def randn(seed, *shape, dtype=F16, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def ints(xs):
    return torch.tensor(xs, dtype=torch.int32, device="cuda")


def over_own(out, want):
    rms = lambda x: float(x.double().pow(2).mean().sqrt())
    return rms(out.double() - want) / rms(want.to(out.dtype).double() - want)


def formula(q, k, v, scale):
    """q [n, H, hd], k, v [L, Hkv, hd], causal at the end of the keys, in 64 bits."""
    n, H, hd = q.shape
    L, g = k.size(0), H // k.size(1)
    kd = k.double().repeat_interleave(g, 1).permute(1, 2, 0).contiguous()
    s = torch.matmul(q.double().transpose(0, 1).contiguous(), kd) * scale
    s = s.masked_fill(torch.arange(L, device="cuda")[None] > torch.arange(n, device="cuda")[:, None] + L - n, -math.inf)
    return torch.matmul(torch.softmax(s, -1), v.double().repeat_interleave(g, 1).transpose(0, 1).contiguous()).transpose(0, 1)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n,L,heads,hd,bound", [
    (30, 600, 4, 128, 1.1), (32, 4000, 8, 64, 1.1), (20, 3000, 4, 256, 1.1),      # few rows: two terms a weight
    (37, 37, 32, 128, 1.1), (130, 130, 8, 128, 1.1), (250, 250, 16, 64, 1.1), (100, 100, 4, 256, 1.1), (200, 200, 4, 32, 1.1),   # short prompts: too
    (512, 512, 32, 128, 1.5), (2600, 2600, 16, 64, 1.5),                          # one term, as documented: 1.2 to 1.4
])
def test_prompt_attention(rk, n, L, heads, hd, bound, dtype):
    q, k, v = randn(1, n, heads, hd, dtype=dtype), randn(2, L, heads, hd, dtype=dtype), randn(3, L, heads, hd, dtype=dtype)
    out = torch.empty_like(q)
    rk.attn_prompt(q, k, v, out, q_start=ints([0, n]), k_start=ints([0]), k_len=ints([L]), timed=False)
    ratio = over_own(out, formula(q, k, v, hd ** -0.5))
    print(f"error {ratio:.3f} times the output's own rounding")
    assert ratio <= bound


@pytest.mark.parametrize("heads,kvh,hd", [(8, 8, 128), (8, 1, 64), (16, 1, 128), (24, 2, 64), (40, 2, 32), (20, 1, 256)])
def test_attention_over_the_4_bit_cache(rk, heads, kvh, hd):
    n, L = 16, 1500
    kc, vc = rk.kv4_cache(n, kvh, L, hd)
    k, v = randn(1, n * L, kvh, hd), randn(2, n * L, kvh, hd)
    pos = torch.zeros(n, dtype=torch.int64, device="cuda")
    rk.kv4_append(k, v, kc, vc, pos, timed=False)
    rk.kv4_read(kc, vc, k, v, timed=False)
    q = randn(3, n, heads, hd)
    out = torch.empty_like(q)
    rk.kv4_attn_decode(q, kc, vc, pos + L - 1, out, timed=False)
    want = torch.cat([formula(q[i:i + 1], k[i * L:(i + 1) * L], v[i * L:(i + 1) * L], hd ** -0.5) for i in range(n)])
    ratio = over_own(out, want)
    print(f"error {ratio:.3f} times the output's own rounding")
    assert ratio <= 1.1


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_token_log_probabilities(rk, dtype):
    """Log probabilities around -10.5, between two powers of two: rounding one is off by 2^-20 / sqrt(12), 2.75e-7, in the mean, a second
    rounding at that size (of the logarithm of the sum) makes it 3.9e-7.  For fp32 logits the difference to the largest, about 2,
    is rounded as well (2^-23 / sqrt(12)).  What else there is: l and t of 512 threads' sums of 68 terms, joined in 15 additions: a
    relative 3e-8, 3e-8 of ln l and about 1e-7 of t / l.  3.2e-7 and 3.5e-7 lie between."""
    rows, vocab = 4096, 35000
    x = randn(5, rows, vocab, dtype=dtype, scale=0.5)
    tokens = torch.randint(0, vocab, (rows,), generator=torch.Generator().manual_seed(6)).cuda()
    lp, en, top, ids = (torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda"), torch.empty(rows, 3, device="cuda"),
                        torch.empty(rows, 3, dtype=torch.int64, device="cuda"))
    rk.token_logprobs(x, tokens, lp, en, top_ids=ids, top_logprobs=top, timed=False)
    squares = torch.zeros(3, dtype=torch.float64, device="cuda")
    for i in range(0, rows, 512):
        logp = torch.log_softmax(x[i:i + 512].double(), -1)
        s = slice(i, i + 512)
        squares[0] += (lp[s].double() - logp.gather(1, tokens[s, None])[:, 0]).pow(2).sum()
        squares[1] += (en[s].double() + (logp.exp() * logp).sum(-1)).pow(2).sum()
        squares[2] += (top[s].double() - logp.gather(1, ids[s])).pow(2).sum() / 3
    errors = (squares / rows).sqrt().tolist()
    print("log probability %.2e, entropy %.2e, alternatives %.2e" % tuple(errors))
    assert errors[0] <= 3.2e-7 and errors[1] <= 3.5e-7 and errors[2] <= 3.2e-7
