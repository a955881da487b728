"""The 4-bit key/value cache (rptc_kernels.kv4_*) against its definition.

Rows: codes, scales and minima bit for bit against the definition in numpy (fp32 quotients, as defined).  Attention: an output
is rounded once (u |o|, u = 2^-11) and every weight once (u A, A = sum p |v| / l, weights below 2^-14 to a multiple of 2^-24 with
the largest at least 1: n 2^-25 max |v|); a score is a sum of hd products and two roundings in fp32, off by at most
E = scale (hd + 4) 2^-24 max sum |q k|, which moves a weight and the sum of weights by factors (together less than 3 E A)."""
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


def randn(seed, *shape, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).half()


def rows_of(x):
    """The cache rows of fp16 vectors [..., hd] (numpy), from the definition."""
    hd = x.shape[-1]
    g = x.astype(np.float32).reshape(x.shape[:-1] + (hd // 32, 32))
    odd = ~np.isfinite(g).all(-1)
    with np.errstate(all="ignore"):
        lo, hi = g.min(-1), g.max(-1)
        s = ((hi - lo) / np.float32(15)).astype(np.float16)
        sf = s.astype(np.float32)[..., None]
        code = np.where(sf > 0, np.clip(np.rint((g - lo[..., None]) / sf), 0, 15), 0)
    code = np.where(odd[..., None], 0, code).astype(np.uint32).reshape(x.shape[:-1] + (hd // 8, 8))
    word = np.zeros(code.shape[:-1], dtype=np.uint32)
    for i in range(8):
        word |= code[..., i] << np.uint32(4 * (i // 2 + 4 * (i % 2)))
    nan = np.float16(np.nan).view(np.uint16) & 0x7E00
    par = np.stack([np.where(odd, nan, s.view(np.uint16)), np.where(odd, nan, lo.astype(np.float16).view(np.uint16))], -1).astype(np.uint16)
    return np.concatenate([np.ascontiguousarray(word).view(np.uint8), np.ascontiguousarray(par.reshape(x.shape[:-1] + (hd // 16,))).view(np.uint8)], -1)


def values_of(rows, hd):
    """What cache rows [..., bytes] stand for, float64 (numpy): fp16(code * s + m)."""
    word = np.ascontiguousarray(rows[..., :hd // 2]).view(np.uint32)
    par = np.ascontiguousarray(rows[..., hd // 2:]).view(np.float16).astype(np.float64).reshape(rows.shape[:-1] + (hd // 32, 2))
    out = np.zeros(rows.shape[:-1] + (hd // 8, 8))
    for i in range(8):
        out[..., i] = (word >> np.uint32(4 * (i // 2 + 4 * (i % 2)))) & 15
    out = out.reshape(rows.shape[:-1] + (hd // 32, 32)) * par[..., :1] + par[..., 1:]
    with np.errstate(all="ignore"):
        return out.astype(np.float16).astype(np.float64).reshape(rows.shape[:-1] + (hd,))


def i64(xs):
    return torch.tensor(xs, dtype=torch.int64, device="cuda")


def i32(xs):
    return torch.tensor(xs, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("heads", [1, 3])
def test_append_writes_the_rows_of_the_definition_and_nothing_else(rk, hd, heads):
    lens, pos, max_len = [5, 0, 1, 17], [3, 0, 10, 0], 20
    total = sum(lens) + 2                                    # two rows behind the last sequence
    k = randn(1, total, heads, hd) * torch.exp(2 * torch.randn(total, heads, 1, device="cuda")).half()
    v = randn(2, total, heads, hd, scale=0.01)
    k[0], k[1, :, :32], k[2, 0, 5], v[3, 0, 7], v[4, 0, 0] = 0.5, 1e-7, float("inf"), float("nan"), 60000.0
    v[4, 0, 1] = -60000.0
    kc, vc = rk.kv4_cache(4, heads, max_len, hd)
    kc.fill_(0xA5)
    vc.fill_(0xA5)
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    ms = rk.kv4_append(k, v, kc, vc, i64(pos), q_start=i32(starts))
    assert ms > 0
    for c, x in ((kc, k), (vc, v)):
        want = np.full(tuple(c.shape), 0xA5, dtype=np.uint8)
        rows = rows_of(x.cpu().numpy())
        for s in range(4):
            for t in range(lens[s]):
                want[s, :, pos[s] + t] = rows[starts[s] + t]
        assert np.array_equal(c.cpu().numpy(), want)
    # read back: the values they stand for, in any layout
    out = torch.full((heads, 4 * max_len, hd), 9.0, dtype=torch.float16, device="cuda").transpose(0, 1)
    outv = torch.full((4 * max_len, heads, 2 * hd), 9.0, dtype=torch.float16, device="cuda")
    kc[kc == 0xA5], vc[vc == 0xA5] = 0, 0                    # (arbitrary bytes may stand for not-a-number)
    rk.kv4_read(kc, vc, out, outv[:, :, :hd], timed=False)
    for got, c in ((out, kc), (outv[:, :, :hd], vc)):
        want = values_of(c.cpu().numpy(), hd).transpose(0, 2, 1, 3).reshape(4 * max_len, heads, hd)
        g = got.cpu().numpy().astype(np.float64)
        assert np.array_equal(np.isnan(g), np.isnan(want)) and np.array_equal(g[~np.isnan(g)], want[~np.isnan(want)])
    assert bool((outv[:, :, hd:] == 9.0).all())


def test_the_error_of_a_row_is_half_a_step(rk):
    x = randn(5, 64, 2, 128)
    kc, vc = rk.kv4_cache(1, 2, 64, 128)
    rk.kv4_append(x, x, kc, vc, i64([0]), timed=False)
    back = torch.empty_like(x)
    rk.kv4_read(kc, vc, back, torch.empty_like(x), timed=False)
    g = x.double().unflatten(2, (4, 32))
    span = (g.amax(-1) - g.amin(-1)).repeat_interleave(32, dim=2)
    # half a step of the rounded scale, the scale's own rounding (15 steps of 2^-11 of it), the value's rounding
    tol = span / 15 * (0.5 + 15 * 2.0 ** -11) + 2.0 ** -11 * x.double().abs().clamp(min=2.0 ** -14) + span * 2.0 ** -11
    assert bool(((back.double() - x.double()).abs() <= tol).all())


def test_positions_outside_the_cache_are_not_written(rk):
    x = randn(6, 12, 2, 64)
    kc, vc = rk.kv4_cache(3, 2, 8, 64)
    kc.fill_(1)
    vc.fill_(1)
    rk.kv4_append(x, x, kc, vc, i64([6, -1, 8]), timed=False)           # four rows each: two fit, none, none
    want = np.full(tuple(kc.shape), 1, dtype=np.uint8)
    want[0, :, 6:8] = rows_of(x[:2].cpu().numpy()).transpose(1, 0, 2)
    assert np.array_equal(kc.cpu().numpy(), want) and np.array_equal(vc.cpu().numpy(), want)
    before = kc.clone()
    rk.kv4_append(x, x, kc, vc, i64([1 << 62, -(1 << 62), 1 << 31]), timed=False)
    rk.kv4_append(x, x, kc, vc, i64([0, 0, 0]), q_start=i32([-(1 << 31), -(1 << 31), 40, 41]), timed=False)
    assert torch.equal(kc, before)


def reference(q, kv, vv, scale):
    """One sequence, one token: q [H, hd], kv, vv [Hkv, L, hd] float64 -> out, tolerance without the output's rounding."""
    g = q.size(0) // kv.size(0)
    kd, vd = kv.repeat_interleave(g, dim=0), vv.repeat_interleave(g, dim=0)
    s = scale * (kd * q[:, None, :]).sum(-1)
    p = torch.softmax(s, dim=-1)
    E = scale * (q.size(1) + 4) * 2.0 ** -24 * (kd.abs() * q[:, None, :].abs()).sum(-1).amax(-1)
    A = (p[..., None] * vd.abs()).sum(1)
    out = (p[..., None] * vd).sum(1)
    return out, (2.0 ** -11 + 3 * E[:, None]) * A + kd.size(1) * 2.0 ** -25 * vd.abs().amax((1, 2))[:, None]


def fill(rk, seqs, heads, max_len, hd, seed=7):
    kc, vc = rk.kv4_cache(seqs, heads, max_len, hd)
    for i in range(0, max_len, 512):
        n = min(512, max_len - i)
        rk.kv4_append(randn(seed + i, seqs * n, heads, hd, scale=1.3), randn(seed + 1 + i, seqs * n, heads, hd), kc, vc, i64([i] * seqs), timed=False)
    return kc, vc


@pytest.mark.parametrize("heads,kvh,hd,max_len,pos", [
    (1, 1, 32, 1, [0]),
    (4, 4, 128, 40, [0, 31, 32, 39]),
    (8, 2, 64, 300, [299, 0, 255, 256, 257]),
    (6, 1, 32, 700, [600, 31]),
    (16, 1, 128, 600, [513]),
    (40, 2, 64, 2100, [2099, 5]),                    # more than 16 query heads a key head, split
    (2, 2, 256, 1200, [1199, 1000]),
    (32, 1, 256, 600, [599]),
    (4, 1, 128, 9000, [8999, 100, 4097]),            # split and joined, pieces without a position
    (32, 32, 128, 1024, [600]),
])
def test_attention_against_the_formula(rk, heads, kvh, hd, max_len, pos):
    n = len(pos)
    kc, vc = fill(rk, n, kvh, max_len, hd)
    q = randn(3, n, heads, hd)
    out = torch.full_like(q, float("nan"))
    assert rk.kv4_attn_decode(q, kc, vc, i64(pos), out) > 0
    for s in range(n):
        L = pos[s] + 1
        kv = torch.from_numpy(values_of(kc[s, :, :L].cpu().numpy(), hd)).cuda()
        vv = torch.from_numpy(values_of(vc[s, :, :L].cpu().numpy(), hd)).cuda()
        want, tol = reference(q[s].double(), kv, vv, hd ** -0.5)
        d = (out[s].double() - want).abs()
        assert bool((d <= tol + 2.0 ** -11 * want.abs() + 2.0 ** -25).all()), (s, float(d.max()))


def test_what_lies_behind_the_position_does_not_count_and_padding_is_left(rk):
    heads, kvh, hd, max_len = 8, 2, 128, 700
    pos = [100, -1, 699, max_len, 0, 1 << 40]
    kc, vc = fill(rk, 6, kvh, max_len, hd)
    q = randn(3, 6, heads, hd)
    out = torch.full_like(q, 3.0)
    rk.kv4_attn_decode(q, kc, vc, i64(pos), out, timed=False)
    assert bool((out[[1, 3, 5]] == 3.0).all()) and not bool((out[[0, 2, 4]] == 3.0).all(-1).any())
    nan = torch.full((1, kvh, hd), float("nan"), dtype=torch.float16, device="cuda")
    for s in (0, 4):
        bad = nan.expand(599, kvh, hd).contiguous()
        rk.kv4_append(bad, bad, kc[s:s + 1], vc[s:s + 1], i64([pos[s] + 1]), timed=False)
    again = torch.full_like(q, 3.0)
    rk.kv4_attn_decode(q, kc, vc, i64(pos), again, timed=False)
    assert torch.equal(out, again)
    # a value that is no number and is seen reaches the heads of its key head, and only those
    bad = randn(1, 1, kvh, hd)
    bad[0, 1, 3] = float("inf")
    rk.kv4_append(randn(2, 1, kvh, hd), bad, kc[:1], vc[:1], i64([50]), timed=False)
    rk.kv4_attn_decode(q, kc, vc, i64(pos), again, timed=False)
    assert bool(torch.isnan(again[0, 4:, :32]).all()) and bool(torch.isfinite(again[0, :4]).all()) and bool(torch.isfinite(again[0, 4:, 32:]).all())


def test_scores_that_rise_along_the_positions(rk):
    hd, L = 64, 900
    k = torch.linspace(-30, 30, L, device="cuda").half()[:, None, None].expand(L, 1, hd).contiguous()
    v = randn(8, L, 1, hd)
    kc, vc = rk.kv4_cache(1, 1, L, hd)
    rk.kv4_append(k, v, kc, vc, i64([0]), timed=False)
    q = torch.ones(1, 2, hd, dtype=torch.float16, device="cuda")
    q[0, 1] = -1
    out = torch.empty_like(q)
    rk.kv4_attn_decode(q, kc, vc, i64([L - 1]), out, scale=0.25, timed=False)
    want, tol = reference(q[0].double(), torch.from_numpy(values_of(kc[0].cpu().numpy(), hd)).cuda(), torch.from_numpy(values_of(vc[0].cpu().numpy(), hd)).cuda(), 0.25)
    assert bool(((out[0].double() - want).abs() <= tol + 2.0 ** -11 * want.abs() + 2.0 ** -25).all())


@pytest.mark.parametrize("heads,kvh,hd", [(4, 4, 64), (8, 2, 128), (2, 1, 32)])
def test_rope_append_is_the_rotation_of_the_fp16_cache_then_append(rk, heads, kvh, hd):
    n, max_len = 3, 50
    g = torch.Generator().manual_seed(1)
    cos, sin = (torch.rand(max_len, hd // 2, generator=g) * 2 - 1).half().cuda(), (torch.rand(max_len, hd // 2, generator=g) * 2 - 1).half().cuda()
    qkv = randn(9, n, (heads + 2 * kvh) * hd)
    pos = i64([7, -1, 49])
    kc, vc = rk.kv4_cache(n, kvh, max_len, hd)
    q_out = torch.full((n, heads, hd), 5.0, dtype=torch.float16, device="cuda")
    rk.kv4_rope_append(qkv, cos, sin, pos, q_out, kc, vc)
    x = qkv.cpu().view(n, heads + 2 * kvh, hd // 2, 2)
    want_k, want_v = rk.kv4_cache(n, kvh, max_len, hd)
    for s, p in ((0, 7), (2, 49)):
        c, sn = cos[p].cpu(), sin[p].cpu()
        a, b = x[s, :, :, 0], x[s, :, :, 1]
        r = torch.stack([a * c - b * sn, a * sn + b * c], dim=-1).reshape(heads + 2 * kvh, hd)       # fp16 throughout
        assert torch.equal(q_out[s].cpu(), r[:heads])
        rk.kv4_append(r[None, heads:heads + kvh].cuda(), qkv[s:s + 1, (heads + kvh) * hd:].reshape(1, kvh, hd), want_k[s:s + 1], want_v[s:s + 1], i64([p]), timed=False)
    assert bool((q_out[1] == 5.0).all()) and torch.equal(kc, want_k) and torch.equal(vc, want_v)


def test_offsets_past_32_bits(rk):
    # a cache of more than 4 GiB: the last sequence's rows lie behind 2^32 bytes
    kvh, hd, max_len, n = 4, 128, 1 << 20, 14
    kc, vc = torch.empty(n, kvh, max_len, 80, dtype=torch.uint8, device="cuda"), torch.empty(n, kvh, max_len, 80, dtype=torch.uint8, device="cuda")
    assert kc.numel() > 1 << 32
    k, v = randn(1, 40, kvh, hd), randn(2, 40, kvh, hd)
    rk.kv4_append(k, v, kc[n - 1:], vc[n - 1:], i64([max_len - 40]), timed=False)
    starts = i32([0] * n + [40])
    kc[n - 1, :, max_len - 40:].zero_()
    rk.kv4_append(k, v, kc, vc, i64([0] * (n - 1) + [max_len - 40]), q_start=starts, timed=False)
    assert np.array_equal(kc[n - 1, :, max_len - 40:].cpu().numpy(), rows_of(k.cpu().numpy()).transpose(1, 0, 2))
    # attend in the last sequence over its first 33 positions and over all (the same row everywhere: its value comes out)
    rk.kv4_append(k[:33], v[:33], kc[n - 1:], vc[n - 1:], i64([0]), timed=False)
    q = randn(3, n, 8, hd)
    out = torch.zeros_like(q)
    rk.kv4_attn_decode(q, kc, vc, i64([-1] * (n - 1) + [32]), out, timed=False)
    want, tol = reference(q[n - 1].double(), torch.from_numpy(values_of(kc[n - 1, :, :33].cpu().numpy(), hd)).cuda(), torch.from_numpy(values_of(vc[n - 1, :, :33].cpu().numpy(), hd)).cuda(), hd ** -0.5)
    assert bool(((out[n - 1].double() - want).abs() <= tol + 2.0 ** -11 * want.abs() + 2.0 ** -25).all()) and not bool(out[:n - 1].any())
    kc[n - 1], vc[n - 1] = kc[n - 1, :, :1].clone(), vc[n - 1, :, :1].clone()
    rk.kv4_attn_decode(q, kc, vc, i64([-1] * (n - 1) + [max_len - 1]), out, timed=False)
    want = torch.from_numpy(values_of(vc[n - 1, :, 0].cpu().numpy(), hd)).cuda().repeat_interleave(2, dim=0)
    # equal weights: p = 1 exactly for every position, so sums and quotient are exact up to fp32 sums of 2^20 terms
    assert bool(((out[n - 1].double() - want).abs() <= 2.0 ** -11 * want.abs() * 1.1 + 2.0 ** -25).all())


def test_the_same_bits_on_another_stream_and_in_two_graphs(rk):
    heads, kvh, hd, max_len = 4, 1, 128, 9000
    kc, vc = fill(rk, 2, kvh, max_len, hd)
    q, pos = randn(3, 2, heads, hd), i64([8000, 77])
    out = torch.empty_like(q)
    rk.kv4_attn_decode(q, kc, vc, pos, out, timed=False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    o2 = torch.empty_like(q)
    with torch.cuda.stream(side):
        rk.kv4_attn_decode(q, kc, vc, pos, o2, timed=False)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, o2)
    graphs, outs = [], []
    for _ in range(2):
        g, o = torch.cuda.CUDAGraph(), torch.zeros_like(q)
        with torch.cuda.graph(g):
            rk.kv4_attn_decode(q, kc, vc, pos, o, timed=False)
        graphs.append(g)
        outs.append(o)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for step in range(3):
        torch.cuda.synchronize()
        with torch.cuda.stream(s1):
            graphs[0].replay()
        with torch.cuda.stream(s2):                             # both at once: a workspace each
            graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], out) and torch.equal(outs[1], out)
        pos.add_(1)
        rk.kv4_attn_decode(q, kc, vc, pos, out, timed=False)


@pytest.mark.parametrize("lens", [[1, 77, 4091, 2000, 513, 2048, 3001, 333, 1024, 3777, 2500, 1666], [4096] * 3 + [5] * 9, [4096, 0, 2049], [600] * 31])
def test_batches_of_unequal_sequences_are_cut_and_joined(rk, lens):
    """The cut is worked out on the device from all lengths together: every sequence comes out as it does alone, within two roundings
    of an output (its pieces, and with them the order of its sums, are others)."""
    heads, kvh, hd, max_len = 8, 2, 64, 4096
    n = len(lens)
    kc, vc = rk.kv4_cache(n, kvh, max_len, hd)
    x = randn(5, n * max_len, kvh, hd)
    rk.kv4_append(x, randn(6, n * max_len, kvh, hd), kc, vc, torch.zeros(n, dtype=torch.int64, device="cuda"))
    q = randn(7, n, heads, hd)
    pos = torch.tensor(lens, device="cuda") - 1
    out = torch.full((n, heads, hd), 7.0, dtype=torch.float16, device="cuda")
    rk.kv4_attn_decode(q, kc, vc, pos, out)
    for i in range(n):
        if lens[i] == 0:
            assert bool((out[i] == 7).all())
            continue
        alone = torch.empty((1, heads, hd), dtype=torch.float16, device="cuda")
        rk.kv4_attn_decode(q[i:i + 1], kc[i:i + 1], vc[i:i + 1], pos[i:i + 1], alone)
        # fp16's step at the output's size, and of sums whose weights (two fp16 terms) and products are rounded at 2^-21 of |v| <= 5
        assert bool(((out[i].double() - alone[0].double()).abs() <= 2.0 ** -10 * alone[0].double().abs() + 2.0 ** -18).all())


def test_more_sequences_than_pieces_wanted(rk):
    # 7 sequences of 128 key heads: more workgroups than compute units from the sequences alone, of a cache long enough to be cut
    seqs, kvh, hd, max_len = 7, 128, 32, 8192
    kc, vc = rk.kv4_cache(seqs, kvh, max_len, hd)
    lens = [8192, 8000, 1, 7000, 0, 8191, 8192]
    g = torch.Generator(device="cuda").manual_seed(3)
    for c in (kc, vc):
        c[..., :hd // 2] = torch.randint(0, 256, c[..., :hd // 2].shape, generator=g, device="cuda", dtype=torch.uint8)
        c[..., hd // 2:] = torch.tensor([0.2, -1.5], dtype=torch.float16, device="cuda").view(torch.uint8)
    q, pos = randn(4, seqs, kvh, hd), torch.tensor(lens, device="cuda") - 1
    out = torch.full((seqs, kvh, hd), 7.0, dtype=torch.float16, device="cuda")
    rk.kv4_attn_decode(q, kc, vc, pos, out)
    for i, n in enumerate(lens):
        if n == 0:
            assert bool((out[i] == 7).all())
            continue
        k, v = (torch.empty((max_len, kvh, hd), dtype=torch.float16, device="cuda") for _ in range(2))
        rk.kv4_read(kc[i:i + 1], vc[i:i + 1], k, v)
        kd, vd = k[:n].double(), v[:n].double()
        s = torch.matmul(kd.transpose(0, 1), q[i].double()[:, :, None])[..., 0] * hd ** -0.5
        p = torch.softmax(s, -1)
        o, A = torch.matmul(p[:, None], vd.transpose(0, 1).contiguous())[:, 0], torch.matmul(p[:, None], vd.abs().transpose(0, 1).contiguous())[:, 0]
        E = hd ** -0.5 * (hd + 4) * 2.0 ** -24 * torch.matmul(kd.abs().transpose(0, 1), q[i].double().abs()[:, :, None]).amax(1)
        tol = 2.0 ** -11 * o.abs() + (2.0 ** -11 + 3 * E) * A + n * 2.0 ** -25 * vd.abs().amax() + 2.0 ** -25
        assert bool(((out[i].double() - o).abs() <= tol).all())


@pytest.mark.parametrize("hd", [32, 128])
def test_codes_beside_the_middle_between_two(rk, hd):
    # groups whose values lie on, and one fp16 step beside, the middles between two codes: the rounded quotient decides
    g = np.random.default_rng(5)
    n = 4096
    lo = g.normal(0, 1, (n, hd // 32, 1)).astype(np.float16).astype(np.float32)
    s = (2.0 ** g.integers(-12, 3, (n, hd // 32, 1))).astype(np.float32) * g.choice([1.0, 1.25, 1.5, 1.0 + 2.0 ** -10], (n, hd // 32, 1)).astype(np.float32)
    x = (lo + s * (g.integers(0, 15, (n, hd // 32, 32)) + 0.5)).astype(np.float16)
    step = g.integers(-1, 2, x.shape)
    x = np.where(step == 0, x, np.nextafter(x, np.where(step > 0, np.float16(np.inf), np.float16(-np.inf)))).astype(np.float16)
    x[..., 0], x[..., 1] = lo[..., 0].astype(np.float16), (lo + 15 * s)[..., 0].astype(np.float16)
    rows = np.ascontiguousarray(x.reshape(n, 1, hd))
    kc, vc = rk.kv4_cache(1, 1, n, hd)
    t = torch.from_numpy(rows).cuda()
    rk.kv4_append(t, t, kc, vc, torch.zeros(1, dtype=torch.int64, device="cuda"))
    want = rows_of(rows.transpose(1, 0, 2))
    assert np.array_equal(kc[0].cpu().numpy(), want) and np.array_equal(vc[0].cpu().numpy(), want)
