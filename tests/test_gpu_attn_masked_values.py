"""rptc_kernels.attn_prompt where V holds values that are no finite numbers: every output element by what its own query sees in its own
dimension, whatever lies in keys that it does not see; elements that see none keep the bits they have without them."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
INF, NAN = float("inf"), float("nan")


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


def attend(rk, q, k, v, lq, lk, causal=True):
    qs, ks = [0], [0]
    for a, b in zip(lq, lk):
        qs.append(qs[-1] + a)
        ks.append(ks[-1] + b)
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
    rk.attn_prompt(q, k, v, out, q_start=ints(qs), k_start=ints(ks[:-1]), k_len=ints(lk), lse=lse, max_k=max(lk), causal=causal, timed=False)
    return out, lse, qs, ks


# lens of queries and of keys, heads, key heads, hd: the forms for few rows (whole and cut), for calls whose longest walk counts (whole and
# cut) and for calls that fill the device
MANY = [1, 0, 127, 128, 129, 33, 300, 2, 64, 65, 31, 96, 7, 260] * 2
FORMS = [([2], [602], 2, 1, 64), ([2], [602], 2, 1, 128), ([5], [600], 4, 2, 256), ([3], [650], 2, 2, 32), ([31], [1500], 2, 2, 128),
         ([2], [4099], 4, 1, 64), ([17], [2500], 2, 1, 256),
         ([512], [512], 32, 32, 128), ([400], [400], 32, 8, 64), ([300], [300], 32, 8, 256), ([400], [400], 32, 8, 32), ([333, 64], [340, 200], 32, 8, 128),
         ([150], [3150], 32, 8, 128), ([300], [5000], 32, 8, 64),
         (MANY, MANY, 32, 8, 64), (MANY, MANY, 32, 8, 128), (MANY, MANY, 32, 8, 256), (MANY, MANY, 32, 8, 32)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lq,lk,heads,kvh,hd", FORMS)
def test_values_that_are_no_numbers_reach_who_sees_them_in_their_dimension(rk, lq, lk, heads, kvh, hd, dtype):
    q, k, v = randn(1, sum(lq), heads, hd, dtype=dtype), randn(2, sum(lk), kvh, hd, dtype=dtype), randn(3, sum(lk), kvh, hd, dtype=dtype)
    clean, clean_lse, qs, ks = attend(rk, q, k, v, lq, lk)
    bad = v.clone()
    for i, n in enumerate(lk):
        # (key, dimension) of a sequence: seen by all or most, by half, by the last few queries
        for back, dim, value in ((n - 1 - n // 60, 0, NAN), (n // 3, 9, INF), (45, 17, -INF), (20, 1, NAN), (2, hd - 1, INF), (1, 5, -INF), (0, 30, NAN)):
            if back < n:
                bad[ks[i + 1] - 1 - back, :, dim] = value
    out, lse, _, _ = attend(rk, q, k, bad, lq, lk)
    assert torch.equal(lse, clean_lse)
    for i in range(len(lq)):
        a, b = slice(qs[i], qs[i + 1]), slice(ks[i], ks[i + 1])
        if not lq[i]:
            continue
        see = torch.arange(lk[i], device="cuda")[None] <= torch.arange(lq[i], device="cuda")[:, None] + lk[i] - lq[i]
        hit = torch.matmul(see.float(), (~torch.isfinite(bad[b])).float().reshape(lk[i], -1)) > 0
        hit = hit.view(lq[i], kvh, hd).repeat_interleave(heads // kvh, 1)
        assert torch.equal(~torch.isfinite(out[a]), hit)
        assert torch.equal(out[a][~hit], clean[a][~hit])


@pytest.mark.parametrize("hd", [64, 128])
def test_one_infinite_value_early_in_a_long_prompt(rk, hd):
    # a value that nearly every query sees, in one dimension: the others keep their bits
    n, heads = 4096, 16
    q, k, v = randn(4, n, heads, hd), randn(5, n, 4, hd), randn(6, n, 4, hd)
    clean, clean_lse, _, _ = attend(rk, q, k, v, [n], [n])
    v[5, 1, 3] = INF
    out, lse, _, _ = attend(rk, q, k, v, [n], [n])
    assert torch.equal(lse, clean_lse) and not bool(torch.isfinite(out[5:, 4:8, 3]).any())
    hit = torch.zeros_like(out, dtype=torch.bool)
    hit[5:, 4:8, 3] = True
    assert torch.equal(out[~hit], clean[~hit])


@pytest.mark.parametrize("lq,lk,heads,kvh,hd", FORMS)
def test_rows_that_see_nothing_of_values_that_are_no_numbers(rk, lq, lk, heads, kvh, hd):
    # more queries than keys, and every value behind the first key not a number: rows in front see nothing, the next one key
    lk = [max(0, n - 3) if len(lk) > 1 else min(n, 3 * lq[0] // 4) for n in lq]
    q, k, v = randn(1, sum(lq), heads, hd), randn(2, sum(lk) + 1, kvh, hd), torch.full((sum(lk) + 1, kvh, hd), NAN, dtype=F16, device="cuda")
    first = 0
    for n in lk:
        if n:
            v[first] = 0.5
        first += n
    out, lse, qs, _ = attend(rk, q, k, v, lq, lk)
    for i, n in enumerate(lq):
        row = torch.arange(n, device="cuda") + lk[i] - n            # the last key a row sees
        o, l = out[qs[i]:qs[i + 1]], lse[qs[i]:qs[i + 1]]
        assert bool((o[row < 0] == 0).all()) and bool((l[row < 0] == -math.inf).all())
        assert bool((o[row == 0] == 0.5).all()) and bool(torch.isfinite(l[row >= 0]).all())
        assert bool(torch.isnan(o[row > 0]).all())
