"""Attention of whole prompts (rptc_kernels.attn_prompt) against the formula in 64 bits.

Tolerance of an output element, from the arithmetic: the output is rounded once (u |o|, u = finfo.eps / 2 of its type) and
every weight p once (u A, A = sum p |v| / l); a score is a sum of hd products and two roundings in fp32, so it is off by at
most E = scale (hd + 4) 2^-24 max sum |q k|, a weight by the factor exp(E) and the sum of weights by another (together less
than 3 E A); fp16 weights below 2^-14 are rounded to a multiple of 2^-24, with the largest weight at least 1 (n 2^-25 max |v|)."""
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


def reference(q, k, v, see, scale):
    """One sequence in 64 bits: q [n, H, hd], k, v [L, Hkv, hd], see [n, L] -> out, lse, the elements' tolerance without the
    output's own rounding, lse's tolerance.  Only what a query sees enters."""
    n, H, hd = q.shape
    out = torch.zeros(n, H, hd, dtype=torch.float64, device=q.device)
    lse = torch.full((n, H), float("-inf"), dtype=torch.float64, device=q.device)
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    u = torch.finfo(q.dtype).eps / 2
    g = H // max(1, k.size(1))
    for h in range(H):
        qd, kd, vd = q[:, h].double(), k[:, h // g].double(), v[:, h // g].double()
        for i in range(n):
            idx = see[i].nonzero().flatten()
            if idx.numel() == 0:
                continue
            s = scale * (kd[idx] @ qd[i])
            E = scale * (hd + 4) * 2.0 ** -24 * float((kd[idx].abs() @ qd[i].abs()).nan_to_num().max())
            lse[i, h] = torch.logsumexp(s, 0)
            p = torch.softmax(s, 0)
            out[i, h] = p @ vd[idx]
            A = p @ vd[idx].abs()
            tol[i, h] = (u + 3 * E) * A + (idx.numel() * 2.0 ** -25 * vd[idx].abs().max() if q.dtype == torch.float16 else 0.0)
            ltol[i, h] = 2 * E + 2.0 ** -21 * (1 + lse[i, h].abs())
    return out, lse, tol, ltol


def visible(lq, lk, causal, device):
    j, i = torch.arange(lk, device=device)[None, :], torch.arange(lq, device=device)[:, None]
    return j <= i + lk - lq if causal else torch.ones(lq, lk, dtype=torch.bool, device=device)


def check(out, lse, want, u_type, rows):
    o, l, tol, ltol = want
    u = torch.finfo(u_type).eps / 2
    got = out[rows].double()
    assert bool(((got - o).abs() <= tol + u * o.abs() + 2.0 ** -25).all()), float(((got - o).abs() - tol - u * o.abs()).max())
    if lse is not None:
        gl = lse[rows].double()
        assert torch.equal(torch.isinf(gl), torch.isinf(l))
        fin = ~torch.isinf(l)
        assert bool(((gl - l).abs()[fin] <= ltol[fin]).all()), float((gl - l).abs()[fin].max())


def randn(seed, *shape, dtype=torch.float16, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def ints(xs):
    return torch.tensor(xs, dtype=torch.int32, device="cuda")


F16, BF16 = torch.float16, torch.bfloat16

CASES = [
    # lens of queries, lens of keys, heads, kv_heads, hd, type, causal
    ([1], [1], 1, 1, 64, F16, True),
    ([1], [130], 4, 2, 128, F16, True),
    ([37], [37], 4, 4, 128, F16, True),
    ([33], [33], 2, 1, 32, BF16, True),
    ([129], [129], 2, 1, 256, F16, True),
    ([65], [65], 2, 2, 256, BF16, False),
    ([64, 1, 0, 63, 128, 2], [64, 1, 0, 63, 128, 2], 4, 2, 64, F16, True),
    ([5, 70, 128, 3], [9, 200, 128, 64], 2, 2, 128, BF16, True),          # chunks at the end of a context
    ([40, 3], [7, 0], 2, 1, 64, F16, True),                              # more queries than keys: the first see nothing
    ([40, 3, 9], [7, 0, 65], 3, 1, 128, F16, False),
    ([257], [300], 2, 2, 64, BF16, True),
    ([31], [1500], 2, 2, 128, F16, True),                                # few rows, many keys: split and joined
    ([2], [4099], 4, 1, 64, BF16, True),
    ([17], [2500], 2, 1, 256, F16, False),
    ([1, 1, 1], [3000, 1, 700], 2, 1, 32, F16, True),
]


@pytest.mark.parametrize("lq,lk,heads,kvh,hd,dtype,causal", CASES)
def test_packed_sequences_against_the_formula(rk, lq, lk, heads, kvh, hd, dtype, causal):
    tq, tk = sum(lq), sum(lk)
    q, k, v = randn(1, tq, heads, hd, dtype=dtype), randn(2, max(tk, 1), kvh, hd, dtype=dtype), randn(3, max(tk, 1), kvh, hd, dtype=dtype)
    out = torch.full_like(q, float("nan"))
    lse = torch.full((tq, heads), float("nan"), device="cuda")
    qs, ks = [0], []
    for a in lq:
        qs.append(qs[-1] + a)
    at = 0
    for b in lk:
        ks.append(at)
        at += b
    ms = rk.attn_prompt(q, k, v, out, q_start=ints(qs), k_start=ints(ks), k_len=ints(lk), causal=causal, lse=lse)
    assert ms > 0
    for s in range(len(lq)):
        rows = slice(qs[s], qs[s + 1])
        want = reference(q[rows], k[ks[s]:ks[s] + lk[s]], v[ks[s]:ks[s] + lk[s]], visible(lq[s], lk[s], causal, "cuda"), hd ** -0.5)
        check(out, lse, want, dtype, rows)


@pytest.mark.parametrize("hd", [64, 128])
def test_layouts_a_projection_and_a_cache_have(rk, hd):
    # q inside [T, (H + 2 Hkv) hd]; k and v a transposed cache with room behind; out a strided buffer too
    H, Hkv, T, past, room = 4, 2, 50, 211, 300
    qkv = randn(4, T, (H + 2 * Hkv) * hd)
    kc, vc = randn(5, Hkv, room, hd), randn(6, Hkv, room, hd)
    kc[:, past + T:], vc[:, past + T:] = float("nan"), float("inf")        # room nobody sees
    q = qkv[:, :H * hd].unflatten(1, (H, hd))
    wide = torch.full((T, H + 1, hd), 7.0, dtype=F16, device="cuda")
    out = wide[:, 1:]
    rk.attn_prompt(q, kc.transpose(0, 1), vc.transpose(0, 1), out, q_start=ints([0, T]), k_start=ints([0]), k_len=ints([past + T]), timed=False)
    want = reference(q, kc.transpose(0, 1)[:past + T], vc.transpose(0, 1)[:past + T], visible(T, past + T, True, "cuda"), hd ** -0.5)
    check(out, None, want, F16, slice(None))
    assert bool((wide[:, 0] == 7.0).all())
    # defaults: one sequence, keys as the queries; another scale; one key head expanded over tokens of equal content
    out2 = torch.empty(T, H, hd, dtype=F16, device="cuda")
    k1 = qkv[:, H * hd:(H + Hkv) * hd].unflatten(1, (Hkv, hd))
    v1 = qkv[:, (H + Hkv) * hd:].unflatten(1, (Hkv, hd))
    rk.attn_prompt(q, k1, v1, out2, scale=0.03, timed=False)
    check(out2, None, reference(q, k1, v1, visible(T, T, True, "cuda"), 0.03), F16, slice(None))
    ke = k1[:1].expand(T, Hkv, hd)
    rk.attn_prompt(q, ke, v1, out2, causal=False, timed=False)
    check(out2, None, reference(q, ke, v1, visible(T, T, False, "cuda"), hd ** -0.5), F16, slice(None))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("lq,lk", [(40, 40), (100, 230), (3, 2000)])
def test_what_a_query_does_not_see_does_not_reach_it(rk, lq, lk, bad):
    # the last two keys hold no numbers: only the last two queries may show it
    H, hd = 2, 64
    q, k, v = randn(7, lq, H, hd), randn(8, lk, H, hd), randn(9, lk, H, hd)
    want = reference(q, k, v, visible(lq, lk, True, "cuda"), hd ** -0.5)
    k[-1], v[-2:] = bad, bad
    out = torch.empty_like(q)
    rk.attn_prompt(q, k, v, out, q_start=ints([0, lq]), k_start=ints([0]), k_len=ints([lk]), timed=False)
    rows = slice(0, lq - 2)
    check(out, None, tuple(t[rows] for t in want), F16, rows)
    tail = out[-1].float()
    assert bool((~torch.isfinite(tail)).all())
    # and a query that holds none stays alone
    k, v = randn(8, lk, H, hd), randn(9, lk, H, hd)
    q2 = q.clone()
    q2[0] = bad
    rk.attn_prompt(q2, k, v, out, q_start=ints([0, lq]), k_start=ints([0]), k_len=ints([lk]), timed=False)
    check(out, None, tuple(t[1:] for t in want), F16, slice(1, None))
    assert bool(torch.isnan(out[0]).all())


def test_large_scores_and_one_dominant_key(rk):
    # scores in the hundreds that rise along the keys (the bound is raised again and again), and fall
    H, hd, n = 2, 64, 300
    q = torch.ones(n, H, hd, dtype=F16, device="cuda")
    v = randn(11, n, H, hd)
    for sign in (1, -1):
        k = (sign * torch.linspace(-40, 40, n, device="cuda"))[:, None, None].expand(n, H, hd).half().contiguous()
        out, lse = torch.empty_like(q), torch.empty(n, H, device="cuda")
        rk.attn_prompt(q, k, v, out, lse=lse, timed=False)
        check(out, lse, reference(q, k, v, visible(n, n, True, "cuda"), hd ** -0.5), F16, slice(None))


def test_rows_of_no_sequence_and_sequences_outside_the_rows_stay(rk):
    H, hd = 2, 64
    q, k, v = randn(12, 200, H, hd), randn(13, 150, H, hd), randn(14, 150, H, hd)
    out = torch.full_like(q, 5.0)
    lse = torch.full((200, H), 5.0, device="cuda")
    # rows 10..60 and 60..90 are sequences; 90..100 has keys past the end, 100..120 a negative start; 120 on: starts past the rows
    rk.attn_prompt(q, k, v, out, q_start=ints([10, 60, 90, 100, 120, 300]), k_start=ints([0, 100, 120, -1, 0]), k_len=ints([50, 50, 31, 20, 10]), lse=lse)
    check(out, lse, reference(q[10:60], k[:50], v[:50], visible(50, 50, True, "cuda"), hd ** -0.5), F16, slice(10, 60))
    check(out, lse, reference(q[60:90], k[100:150], v[100:150], visible(30, 50, True, "cuda"), hd ** -0.5), F16, slice(60, 90))
    for rows in (slice(0, 10), slice(90, 200)):
        assert bool((out[rows] == 5.0).all()) and bool((lse[rows] == 5.0).all())


def test_many_short_sequences(rk):
    # more sequences than a wave looks up at once
    H, hd, n = 1, 64, 150
    g = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 6, (n,), generator=g).tolist()
    starts = [0]
    for a in lens:
        starts.append(starts[-1] + a)
    q, k, v = (randn(s, starts[-1], H, hd) for s in (1, 2, 3))
    out = torch.empty_like(q)
    rk.attn_prompt(q, k, v, out, q_start=ints(starts), timed=False)
    for s in range(n):
        rows = slice(starts[s], starts[s + 1])
        if lens[s]:
            check(out, None, reference(q[rows], k[rows], v[rows], visible(lens[s], lens[s], True, "cuda"), hd ** -0.5), F16, rows)


def test_the_same_bits_again_on_another_stream_and_in_a_graph(rk):
    H, hd = 4, 128
    q, k, v = randn(21, 30, H, hd), randn(22, 1900, H, hd), randn(23, 1900, H, hd)      # split over its keys: a workspace
    args = dict(q_start=ints([0, 30]), k_start=ints([0]), k_len=ints([1900]), timed=False)
    out = torch.empty_like(q)
    rk.attn_prompt(q, k, v, out, **args)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out2 = torch.empty_like(q)
    with torch.cuda.stream(side):
        rk.attn_prompt(q, k, v, out2, **args)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, out2)
    outs, graphs = [], []
    for _ in range(2):
        g, o = torch.cuda.CUDAGraph(), torch.zeros_like(q)
        with torch.cuda.graph(g):
            rk.attn_prompt(q, k, v, o, **args)
        graphs.append(g)
        outs.append(o)
    for _ in range(3):
        for g, o in zip(graphs, outs):
            o.zero_()
            g.replay()
        torch.randn(1 << 20, device="cuda").sum()                       # the program's own work in between
        torch.cuda.synchronize()
        assert torch.equal(outs[0], out) and torch.equal(outs[1], out)
    q.mul_(0.5)                                                         # new contents, old graph
    rk.attn_prompt(q, k, v, out, **args)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], out)
