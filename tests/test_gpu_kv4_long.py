"""rptc_kernels.kv4_attn_decode over caches of very many positions."""
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


def randn(seed, *shape):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").half()


def i64(xs):
    return torch.tensor(xs, dtype=torch.int64, device="cuda")


def test_pieces_of_more_than_four_gib_behind_a_tile(rk):
    """The most positions a cache may have, in pieces of 2^25: tiles so far in front of a piece's end that the bytes between pass
    2^32.  A key that outweighs all others (score 240 against 0: every other weight is below 2^-300) in the tile for which
    that distance is 2^32 and 1024 bytes: its value comes out, to the output's rounding, which the value, an fp16, does not have."""
    heads, hd, max_len, row = 1024, 256, 1 << 26, 160
    kc, vc = rk.kv4_cache(2, 1, max_len, hd)
    ends = [1 << 25, 1 << 26]
    at = [end - ((1 << 32) + 1024) // row + 20 for end in ends]
    values = randn(1, 4, 1, hd)
    for i, p in enumerate(at):
        k = torch.zeros(2, 1, hd, dtype=torch.float16, device="cuda")
        k[:, 0, 32 * i] = 30.0
        rk.kv4_append(k, values[2 * i:2 * i + 2], kc, vc, i64([p, p]), timed=False)
    q = torch.zeros(2, heads, hd, dtype=torch.float16, device="cuda")
    q[:, 0::2, 0], q[:, 1::2, 32] = 8.0, 8.0
    out = torch.empty_like(q)
    rk.kv4_attn_decode(q, kc, vc, i64([max_len - 1, max_len - 1]), out, scale=1.0, timed=False)
    want = torch.empty_like(values)
    cache = rk.kv4_cache(4, 1, 1, hd)
    rk.kv4_append(values, values, *cache, i64([0] * 4), timed=False)
    rk.kv4_read(*cache, torch.empty_like(values), want, timed=False)
    for s in range(2):
        for i in range(2):
            assert torch.equal(out[s, i::2], want[2 * i + s].expand(heads // 2, hd)), (s, i)


@pytest.mark.parametrize("heads,kvh,seqs", [(4, 4, 256), (32, 2, 512)])
def test_many_weights_far_below_the_largest(rk, heads, kvh, seqs):
    """A key in front that outweighs each other one by 2^26, as the first token of a trained model's context may, with a value of 0, and
    values of 1 behind it: the output is what the others weigh together, (n - 1) / (2^26 + n - 1).  The scores are hd (exact) and 0, the
    scale makes the one 26 ln 2 to 26 * 2^-23.  An fp16 weight is a multiple of 2^-24; with the largest at 2^7 at least, the
    others are 32 of those.  Tolerance: the output's half step, the scores' fp32 roundings (E = 18.1 (hd + 4) 2^-24, 3 E of the output),
    fp32 sums of 2^11 terms behind each other (2^-13)."""
    hd, n = 64, 16384
    kc, vc = rk.kv4_cache(seqs, kvh, n, hd)
    par = torch.tensor([0.0, 1.0], dtype=torch.float16, device="cuda").view(torch.uint8).repeat(hd // 32)      # scale 0, minimum 1
    kc[:, :, 0, hd // 2:], vc[:, :, 1:, hd // 2:] = par, par
    q = torch.ones(seqs, heads, hd, dtype=torch.float16, device="cuda")
    out = torch.empty_like(q)
    rk.kv4_attn_decode(q, kc, vc, i64([n - 1] * seqs), out, scale=26 * math.log(2) / hd, timed=False)
    rest = (n - 1) * 2.0 ** -26
    want = rest / (1 + rest)
    assert bool(((out.double() - want).abs() <= want * (2.0 ** -11 + 3 * 18.1 * (hd + 4) * 2.0 ** -24 + 2.0 ** -13) + 2.0 ** -25).all()), (want, float(out.min()), float(out.max()))


@pytest.mark.parametrize("hd,L", [(64, 131072), (128, 140001)])
def test_one_key_head_in_as_many_pieces_as_are_joined(rk, hd, L):
    """One long sequence of one key head, cut into as many pieces as are joined, against the formula in 64 bits.  Tolerance: the
    output's rounding (u |o|, u = 2^-11), the weights' in two fp16 terms (2^-21 A, A = sum p |v|), the scores' (E = scale (hd + 4)
    2^-24 max sum |q k|, 3 E A), and fp32 sums of n positive terms in groups of at most 2^10 behind each other (2^-13 A)."""
    heads, most = 4, 128                                      # room for as many pieces as there can be, no more workgroups than these
    assert rk.library().rptc_kv4_attn_decode_workspace_bytes(1, heads, 1, hd, L) <= heads * most * (hd + 2) * 4
    kc, vc = rk.kv4_cache(1, 1, L, hd)
    k, v = randn(1, L, 1, hd), randn(2, L, 1, hd)
    rk.kv4_append(k, v, kc, vc, i64([0]), timed=False)
    rk.kv4_read(kc, vc, k, v, timed=False)
    q = randn(3, 1, heads, hd)
    for pos in (L - 1, L - 77, 40000):
        out = torch.empty_like(q)
        rk.kv4_attn_decode(q, kc, vc, i64([pos]), out, timed=False)
        kd, vd, qd = k[:pos + 1, 0].double(), v[:pos + 1, 0].double(), q[0].double()
        p = torch.softmax(qd @ kd.t().contiguous() * hd ** -0.5, -1)
        o, A = p @ vd, p @ vd.abs()
        E = hd ** -0.5 * (hd + 4) * 2.0 ** -24 * (qd.abs() @ kd.abs().t().contiguous()).amax(-1, keepdim=True)
        assert bool(((out[0].double() - o).abs() <= 2.0 ** -11 * o.abs() + (2.0 ** -21 + 3 * E + 2.0 ** -13) * A + 2.0 ** -25).all()), pos


@pytest.mark.parametrize("heads,kvh,hd,n", [(4, 4, 64, 700), (32, 2, 128, 700), (8, 1, 128, 9001), (2, 2, 256, 5000), (3, 3, 32, 900)])
def test_scores_of_millions_and_more(rk, heads, kvh, hd, n):
    """Scores of up to 2^34, 2^23 and more apart: one position takes all weight, or those equal to it share it.  The output is the mean
    of their values, rounded: each weight is 1, up to roundings of the sum and the quotient, 2^-20."""
    g = torch.Generator(device="cuda").manual_seed(5)
    level = torch.randperm(n, generator=g, device="cuda") // 3
    k = (12 * (level - n // 6))[:, None, None].half().expand(n, kvh, hd).contiguous()       # one value a row: held exactly, as its minimum
    level = k[:, 0, 0].double()
    v = randn(8, n, kvh, hd)
    kc, vc = rk.kv4_cache(1, kvh, n, hd)
    rk.kv4_append(k, v, kc, vc, i64([0]), timed=False)
    rk.kv4_read(kc, vc, k, v, timed=False)
    assert torch.equal(k[:, 0, 0].double(), level)
    q = torch.full((1, heads, hd), 60000.0, dtype=torch.float16, device="cuda")
    q[0, 1::2] *= -1
    for pos in (n - 1, n // 2, 40):
        out = torch.empty_like(q)
        rk.kv4_attn_decode(q, kc, vc, i64([pos]), out, timed=False)
        vd = v[:pos + 1].double().repeat_interleave(heads // kvh, 1)
        for h in range(heads):
            seen = level[:pos + 1] * (-1 if h % 2 else 1)
            want = vd[seen == seen.max(), h].mean(0)
            assert bool(((out[0, h].double() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -20).all()), (pos, h)
