"""Rows of the 4-bit cache (rptc_kernels.kv4_append) at the ends of fp16's range."""
import numpy as np
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


def groups():
    """Groups of 32 finite values: largest and smallest from the ends of the range, zero, the smallest numbers and between."""
    ends = [65504.0, 65472.0, 60000.0, 32768.0, 1.0, 2.0 ** -14, 2.0 ** -24, 0.0]
    ends = np.array(sorted({s * e for e in ends for s in (1, -1)}), dtype=np.float16)
    g = np.random.default_rng(7)
    out = []
    for hi in ends:
        for lo in ends[ends <= hi]:
            x = (lo.astype(np.float64) + (hi.astype(np.float64) - lo) * g.random(32)).astype(np.float16)
            x[3], x[17] = hi, lo
            out.append(x + np.float16(0))                     # (no zeros of a sign)
    return np.stack(out)


def steps_of(g):
    """Scale, minimum and codes of groups [n, 32], from the definition."""
    x = g.astype(np.float32)
    lo, hi = x.min(-1), x.max(-1)
    s = ((hi - lo) / np.float32(15)).astype(np.float16)
    with np.errstate(over="ignore"):
        above = np.isinf((15.0 * s.astype(np.float64) + lo).astype(np.float16))
    s = np.where(above, np.nextafter(s, np.float16(0)), s).astype(np.float16)
    sf = s.astype(np.float32)[:, None]
    with np.errstate(all="ignore"):
        code = np.where(sf > 0, np.clip(np.rint((x - lo[:, None]) / sf), 0, 15), 0)
    return s, lo, code


def test_finite_values_stay_finite(rk):
    """A value comes back within half a step, 15 of the scale's roundings (down, where 15 s + m would be infinite: up to a whole unit in
    the last place, 2^-10 of it, or the smallest number) and its own."""
    g = groups()
    x = torch.from_numpy(g).cuda().view(-1, 1, 32)
    n = x.size(0)
    kc, vc = rk.kv4_cache(1, 1, n, 32)
    rk.kv4_append(x, x, kc, vc, torch.zeros(1, dtype=torch.int64, device="cuda"), timed=False)
    k, v = torch.empty_like(x), torch.empty_like(x)
    rk.kv4_read(kc, vc, k, v, timed=False)
    s, lo, code = steps_of(g)
    assert torch.equal(k, v) and bool(torch.isfinite(k).all())
    want = (code * s.astype(np.float64)[:, None] + lo[:, None]).astype(np.float16)
    assert np.array_equal(k[:, 0].cpu().numpy(), want)
    wide = g.astype(np.float64)
    span = wide.max(-1) - wide.min(-1)
    unit = np.maximum(span / 15 * 2.0 ** -10, 2.0 ** -24)
    bound = span / 30 + 15.5 * unit + np.maximum(np.abs(wide).max(-1) * 2.0 ** -11, 2.0 ** -25)
    assert (np.abs(k[:, 0].cpu().numpy().astype(np.float64) - wide) <= bound[:, None]).all()


def test_one_token_on_its_way_into_the_cache(rk):
    # the same rows by the fused rotation and append (angle 0: cos 1, sin 0 leave q and k as they are), and attention over one of them
    g = torch.from_numpy(groups()).cuda()
    n, hd = g.size(0) // 4, 128
    rows = g[:4 * n].reshape(n, 1, hd)
    cos, sin = torch.ones(1, hd // 2, dtype=torch.float16, device="cuda"), torch.zeros(1, hd // 2, dtype=torch.float16, device="cuda")
    pos = torch.zeros(n, dtype=torch.int64, device="cuda")
    a, b = rk.kv4_cache(n, 1, 1, hd), rk.kv4_cache(n, 1, 1, hd)
    rk.kv4_append(rows, rows, *a, pos, timed=False)
    q = torch.empty(n, 1, hd, dtype=torch.float16, device="cuda")
    rk.kv4_rope_append(torch.cat([torch.zeros_like(rows), rows, rows], 1).reshape(n, 3 * hd), cos, sin, pos, q, *b, timed=False)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    k, v, out = torch.empty_like(rows), torch.empty_like(rows), torch.empty_like(rows)
    rk.kv4_read(*a, k, v, timed=False)
    rk.kv4_attn_decode(q, *a, pos, out, timed=False)                      # one position: its value, to a rounding
    assert bool(torch.isfinite(out).all()) and bool(((out.double() - v.double()).abs() <= 2.0 ** -11 * v.double().abs() + 2.0 ** -25).all())
