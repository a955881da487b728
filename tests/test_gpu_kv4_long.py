"""rptc_kernels.kv4_attn_decode over caches of very many positions."""
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
