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
