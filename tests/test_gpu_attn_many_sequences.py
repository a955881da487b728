"""rptc_kernels.attn_prompt over calls of very many sequences, whose tiles are found through a table."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F16 = torch.float16


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


def ints(xs):
    return torch.tensor(xs, dtype=torch.int32, device="cuda")


def lengths(n, most, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, most + 1, (n,), generator=g).tolist()


@pytest.mark.parametrize("n,most,heads,kvh,hd,seed", [(129, 40, 4, 1, 64, 6), (257, 3, 1, 1, 64, 1), (1000, 70, 2, 1, 64, 2), (1025, 200, 4, 2, 32, 3), (5000, 9, 2, 2, 128, 4), (300, 300, 32, 8, 64, 5)])
def test_each_sequence_gets_what_it_has_in_a_call_of_few(rk, n, most, heads, kvh, hd, seed):
    """Sequences of the packed call against calls of at most 100 sequences each (found without a table, tested elsewhere against the
    formula), to the output's rounding and the weights' (u (|o| + A) with A <= max |v|; another form may take them)."""
    lens = lengths(n, most, seed)
    starts = [0]
    for a in lens:
        starts.append(starts[-1] + a)
    T = starts[-1]
    q, k, v = randn(1, T + 5, heads, hd), randn(2, T + 5, kvh, hd), randn(3, T + 5, kvh, hd)
    out, lse = torch.full_like(q, 7.0), torch.full((T + 5, heads), 7.0, device="cuda")
    # starts of the keys given, not as the queries': shifted by five rows
    ks = [s + 5 for s in starts[:-1]]
    rk.attn_prompt(q, k, v, out, q_start=ints(starts), k_start=ints(ks), k_len=ints(lens), lse=lse, max_k=max(lens), timed=False)
    assert bool((out[T:] == 7).all()) and bool((lse[T:] == 7).all())
    again, lse2 = torch.full_like(out, 7.0), torch.full_like(lse, 7.0)
    for i in range(0, n, 100):
        j = min(n, i + 100)
        rk.attn_prompt(q, k, v, again, q_start=ints(starts[i:j + 1]), k_start=ints(ks[i:j]), k_len=ints(lens[i:j]), lse=lse2, max_k=max(lens), timed=False)
    bound = 2 * 2.0 ** -11 * (again.double().abs() + float(v.abs().max()))
    assert bool(((out.double() - again.double()).abs() <= bound).all())
    assert bool(((lse - lse2).abs() <= 2.0 ** -19 * (1 + lse2.abs())).all())


def test_cut_and_joined(rk):
    # few queries of each of 300 sequences, one of them behind very many keys: pieces, and rows found again by the join
    n, heads, hd = 300, 4, 64
    lens = [i % 3 for i in range(n)]
    lens[123] = 2
    starts = [0]
    for a in lens:
        starts.append(starts[-1] + a)
    L = 9000
    q, k, v = randn(1, starts[-1], heads, hd), randn(2, L, 1, hd), randn(3, L, 1, hd)
    klen = [L if i == 123 else 40 for i in range(n)]
    out = torch.full_like(q, 7.0)
    for max_k in (L, None, 100):                  # (an upper bound of k_len, all keys, and one that is wrong: it only picks the form)
        rk.attn_prompt(q, k, v, out, q_start=ints(starts), k_start=ints([0] * n), k_len=ints(klen), max_k=max_k, timed=False)
        for i in (0, 1, 2, 122, 123, 124, 298, 299):
            rows = slice(starts[i], starts[i + 1])
            if not lens[i]:
                continue
            s = torch.matmul(q[rows].double().transpose(0, 1), k[:klen[i], 0].double().t().contiguous()) * hd ** -0.5
            see = torch.arange(klen[i], device="cuda")[None] <= torch.arange(lens[i], device="cuda")[:, None] + klen[i] - lens[i]
            p = torch.softmax(s.masked_fill(~see, -math.inf), -1)
            o, A = torch.matmul(p, v[:klen[i], 0].double()), torch.matmul(p, v[:klen[i], 0].double().abs())
            # one rounding of the output and of each weight, scores to 2^-16 (sums of 64 products of about 1, 2^-24 each and its order)
            assert bool(((out[rows].double().transpose(0, 1) - o).abs() <= 2.0 ** -11 * o.abs() + (2.0 ** -11 + 2.0 ** -14) * A + 2.0 ** -25).all())


def test_sequences_that_are_none(rk):
    # among 700: starts that fall, lie in front of or behind the rows, keys that do not exist; the others are what they are without these
    n, heads, hd = 700, 2, 64
    lens = [5] * n
    starts = [5 * i for i in range(n + 1)]
    T = starts[-1]
    q, k, v = randn(1, T, heads, hd), randn(2, T, heads, hd), randn(3, T, heads, hd)
    clean, out = torch.full_like(q, 7.0), torch.full_like(q, 7.0)
    args = dict(k_start=ints(starts[:-1]), timed=False)
    rk.attn_prompt(q, k, v, clean, q_start=ints(starts), k_len=ints(lens), **args)
    bad = list(starts)
    bad[100], bad[200], bad[300], bad[350] = -7, T + 1, 1 << 30, -(1 << 31)
    klen = list(lens)
    klen[500], klen[600] = -1, T
    rk.attn_prompt(q, k, v, out, q_start=ints(bad), k_len=ints(klen), **args)
    left = torch.zeros(T, dtype=torch.bool, device="cuda")
    for i in (99, 100, 199, 200, 299, 300, 349, 350, 500, 600):
        left[5 * i:5 * i + 5] = True
    assert bool((out[left] == 7).all()) and torch.equal(out[~left], clean[~left])


def test_as_many_sequences_as_a_call_takes(rk):
    """2^20 sequences of one row and one key each: the output is the key's value, exactly."""
    n, hd = 1 << 20, 32
    q, v = randn(1, n, 1, hd), randn(2, n, 1, hd)
    out = torch.empty_like(q)
    rk.attn_prompt(q, q, v, out, q_start=torch.arange(n + 1, dtype=torch.int32, device="cuda"), max_k=1, timed=False)
    assert torch.equal(out, v)


def test_two_graphs(rk):
    n, heads, hd = 400, 2, 64
    starts = torch.arange(0, 4 * n + 1, 4, dtype=torch.int32, device="cuda")
    q, k, v = randn(1, 4 * n, heads, hd), randn(2, 4 * n, heads, hd), randn(3, 4 * n, heads, hd)
    out, graphs, outs = torch.empty_like(q), [], []
    rk.attn_prompt(q, k, v, out, q_start=starts, max_k=8, timed=False)
    for _ in range(2):
        g, o = torch.cuda.CUDAGraph(), torch.zeros_like(q)
        with torch.cuda.graph(g):
            rk.attn_prompt(q, k, v, o, q_start=starts, max_k=8, timed=False)
        graphs.append(g)
        outs.append(o)
    for step in range(3):
        for g, o in zip(graphs, outs):
            o.zero_()
            g.replay()
        torch.randn(1 << 16, device="cuda").sum()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], out) and torch.equal(outs[1], out)
        starts[1:-1] += 1                                       # other sequences, the same graphs
        rk.attn_prompt(q, k, v, out, q_start=starts, max_k=8, timed=False)
