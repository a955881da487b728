"""The prompt attention, the 4-bit cache and the token log probabilities together, as the decoder and the perplexity harness run
them: every operator's result inside the model against 64-bit arithmetic on what the model handed it."""
import math

import pytest
import torch

from rptc_kernels import eval_ppl
from rptc_kernels.llama_decode import LlamaShape, QuantizedLlama, greedy_decode

pytestmark = pytest.mark.gpu

U = 2.0 ** -11          # half a step of fp16


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


def attention(q, k, v, first):
    """64-bit attention of rows q [T, heads, hd], row t seeing keys 0 .. first + t of k, v [n, heads, hd], and the bound on what
    roundings may add: one of the output (U |o|), one of every weight (U A, A the sum of weight * |v|; weights below 2^-14 to
    multiples of 2^-24 against a largest one of at least 1, n 2^-25 max |v|), and scores summed in fp32 (hd + 4 steps of
    2^-24 of the sum of |q k|, which moves weights and their sum: 3 E A)."""
    q, k, v = q.double(), k.double(), v.double()
    T, n, hd = q.size(0), k.size(0), q.size(2)
    s = torch.matmul(q.transpose(0, 1), k.permute(1, 2, 0).contiguous()) * hd ** -0.5
    most = torch.matmul(q.abs().transpose(0, 1), k.abs().permute(1, 2, 0).contiguous()) * hd ** -0.5
    seen = torch.arange(n, device=q.device)[None] <= first + torch.arange(T, device=q.device)[:, None]
    p = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
    o = torch.matmul(p, v.transpose(0, 1).contiguous())
    A = torch.matmul(p, v.abs().transpose(0, 1).contiguous())
    E = (hd + 4) * 2.0 ** -24 * most.masked_fill(~seen, 0).amax(-1, keepdim=True)
    bound = U * o.abs() + (U + 3 * E) * A + n * 2.0 ** -25 * v.abs().amax() + 2.0 ** -25
    return o.transpose(0, 1), bound.transpose(0, 1)


def check(out, want):
    o, bound = want
    err = (out.double() - o).abs()
    assert bool((err <= 1.01 * bound).all()), float((err / bound).max())


def test_packed_prompts_layer_by_layer_and_against_one_at_a_time(rk, monkeypatch):
    """Every attention call of a packed pass within its rounding bound; the logits those of each prompt alone in chunks.

    Logits: two paths of about ten fp16 roundings a layer each, U / sqrt(3) of the value a rounding in the mean: 1.3e-3 a layer,
    1.8e-3 for two; 1e-2 leaves a factor of 5."""
    shape = LlamaShape(layers=2, d_model=256, heads=4, d_ff=704, vocab=1000, max_len=128)
    model = QuantizedLlama(shape, S=8, seed=7)
    lens = [40, 1, 128, 33]
    tokens = torch.randint(0, shape.vocab, (sum(lens),), generator=torch.Generator().manual_seed(1)).cuda()
    calls = []
    plain = rk.attn_prompt
    monkeypatch.setattr(rk, "attn_prompt", lambda q, k, v, out, **kw: calls.append((q, k, v, out)) or plain(q, k, v, out, **kw))
    with torch.no_grad():
        logits = model.forward_prompt(tokens, lens, all_logits=True)
        last = model.forward_prompt(tokens, lens)
    assert len(calls) == 2 * shape.layers and logits.shape == (sum(lens), shape.vocab) and last.shape == (len(lens), shape.vocab)
    for q, k, v, out in calls:
        for i, n in enumerate(lens):
            rows = slice(sum(lens[:i]), sum(lens[:i]) + n)
            check(out[rows], attention(q[rows], k[rows], v[rows], 0))
    monkeypatch.undo()
    for i, n in enumerate(lens):
        start = sum(lens[:i])
        pos = torch.arange(n, device="cuda")
        with torch.no_grad():
            for p0 in range(0, n, 32):
                want = model.forward_tokens(tokens[start + p0:start + p0 + 32][:n - p0], pos[p0:p0 + 32], all_logits=True)
                got = logits[start + p0:start + p0 + want.size(0)]
                assert float((got - want).norm() / want.norm()) < 1e-2
        assert float((last[i] - logits[start + n - 1]).norm() / last[i].norm()) < 1e-2


@pytest.mark.parametrize("shape", [LlamaShape(layers=2, d_model=256, heads=4, d_ff=704, vocab=1000, max_len=128),
                                   LlamaShape(layers=2, d_model=256, heads=2, d_ff=704, vocab=1000, max_len=4099)],
                         ids=["hd 64", "hd 128, cut sequences"])
def test_decoder_on_a_4_bit_cache(rk, monkeypatch, shape):
    """Prompt into the cache, then tokens: the rows in the cache stand for the rotated keys to half a code step, the attention of every layer
    is that over the values the cache stands for, a replayed graph decodes the tokens that launches decode."""
    model = QuantizedLlama(shape, S=8, seed=7, cache_bits=4)
    H, hd = shape.heads, shape.head_dim
    prompt = torch.randint(0, shape.vocab, (77,), generator=torch.Generator().manual_seed(3))
    runs = {}
    for mode in ("fused_graph", "fused", "glue_graph", "glue", "torch"):
        for c in (*model.k_cache, *model.v_cache):
            c.fill_(0xFF)                       # rows never written read as not-a-number: nothing may see them
        runs[mode], _ = greedy_decode(model, prompt, 12, mode=mode, whole_prompt=mode != "glue")
        assert all(0 <= t < shape.vocab for t in runs[mode])
    assert runs["fused_graph"] == runs["fused"] and runs["glue_graph"][0] == runs["torch"][0]

    calls = []
    append, decode = rk.kv4_append, rk.kv4_attn_decode
    monkeypatch.setattr(rk, "kv4_append", lambda k, v, kc, vc, pos, **kw: calls.append((k.clone(), v.clone(), kc, vc)) or append(k, v, kc, vc, pos, **kw))
    with torch.no_grad():
        model.forward_prompt(prompt.cuda(), store=True)
    n = prompt.numel()
    assert len(calls) == shape.layers
    for i, (k, v, kc, vc) in enumerate(calls):
        ks, vs = (torch.empty((n, H, hd), dtype=torch.float16, device="cuda") for _ in range(2))
        rk.kv4_read(kc, vc, ks, vs)
        for x, y in ((k, ks), (v, vs)):
            x, y = x.double().view(n, H, hd // 32, 32), y.double().view(n, H, hd // 32, 32)
            top, low = x.amax(-1, keepdim=True), x.amin(-1, keepdim=True)
            # half a step; the step itself rounded to fp16 (U of it, 15 times, subnormal steps by 2^-25); the value once more
            step = (top - low) / 15
            bound = step / 2 * (1 + 2.0 ** -10) + 15 * (U * step + 2.0 ** -25) + U * y.abs() + 2.0 ** -25
            assert bool(((x - y).abs() <= bound).all())
    monkeypatch.undo()

    # one more token: the attention of each layer from what the step left in its buffers and its cache
    seen = []

    def watch(q, kc, vc, pos, out, **kw):
        decode(q, kc, vc, pos, out, **kw)
        seen.append((q.clone(), kc, vc, out.clone()))
    monkeypatch.setattr(rk, "kv4_attn_decode", watch)
    with torch.no_grad():
        logits = model.decode_step(torch.tensor([5], device="cuda"), torch.tensor([n], device="cuda"))
        chunk = model.forward_tokens(torch.tensor([5], device="cuda"), torch.tensor([n], device="cuda"))
    assert len(seen) == 2 * shape.layers
    for q, kc, vc, out in seen:
        ks, vs = (torch.empty((n + 1, H, hd), dtype=torch.float16, device="cuda") for _ in range(2))
        rk.kv4_read(kc, vc, ks, vs)
        check(out, attention(q, ks, vs, n))
    assert bool(torch.isfinite(logits).all()) and float((logits - chunk).norm() / chunk.norm()) < 5e-2


def test_scores_of_packed_texts(rk):
    """score_tokens: log probabilities, entropies and alternatives of the pass's own logits to fp32's accuracy; the last token of each text scores
    nothing.  packed_perplexity: a token's log probability moves by at most twice the largest difference of two paths' logits."""
    shape = LlamaShape(layers=2, d_model=256, heads=4, d_ff=704, vocab=1000, max_len=64)
    model = QuantizedLlama(shape, S=8, seed=11)
    tokens = torch.as_tensor(eval_ppl.synthetic_tokens(3 * 64 + 5, shape.vocab, seed=5), dtype=torch.int64)
    lens = [64, 1, 63, 64, 5]
    with torch.no_grad():
        logits = model.forward_prompt(tokens.cuda(), lens, all_logits=True, half_logits=True)
    got = eval_ppl.score_tokens(model, tokens, lens, top=5)
    logp = torch.log_softmax(logits.double(), -1)
    ends = (torch.tensor(lens).cumsum(0) - 1).cuda()
    inner = torch.ones(tokens.numel(), dtype=torch.bool, device="cuda")
    inner[ends] = False
    want = logp[:-1].gather(1, tokens.cuda()[1:, None])[:, 0]
    # a sum of 1000 exponentials (each to 2^-20 of itself at these sizes) and its logarithm, about 20 in all
    assert bool(torch.isnan(got["logprob"][ends]).all())
    assert float((got["logprob"][:-1].double() - want)[inner[:-1]].abs().max()) < 2e-5
    assert float((got["entropy"].double() + (logp.exp() * logp).sum(-1)).abs().max()) < 1e-4
    assert torch.equal(got["top_logprobs"], got["top_logprobs"].sort(-1, descending=True).values)
    assert float((got["top_logprobs"].double() - logp.topk(5).values).abs().max()) < 2e-5
    assert torch.equal(logits.gather(1, got["top_ids"]), logits.topk(5).values)

    windows = tokens[:192]
    ppl, loss, n = eval_ppl.packed_perplexity(model, windows, 64, windows_per_pass=2)
    ppl_c, loss_c, n_c = eval_ppl.perplexity(eval_ppl.llama_logits_fn(model), windows, 64)
    logits_fn = eval_ppl.llama_logits_fn(model)
    with torch.no_grad():
        apart = max(float((model.forward_prompt(w.cuda(), all_logits=True) - logits_fn(w).cuda().view(64, -1)).abs().max())
                    for w in windows.view(3, 64))
    assert n == n_c == 3 and abs(loss - loss_c) <= 2 * apart + 1e-4 and apart < 0.1
    assert ppl == math.exp(loss)
