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


def test_two_threads_on_two_streams_at_once(rk):
    """Calls that overlap have a workspace each: split attention, cut decode attention and scores from two threads, every result the
    bits that the call gives alone."""
    import threading
    g = torch.Generator(device="cuda").manual_seed(9)
    rand = lambda *shape: torch.randn(shape, generator=g, device="cuda").half()
    jobs = []
    for n, past in ((7, 2500), (30, 4000)):
        q, k, v = rand(n, 4, 64), rand(past, 2, 64), rand(past, 2, 64)
        jobs.append((lambda out, q=q, k=k, v=v: rk.attn_prompt(q, k, v, out, timed=False), q.shape, torch.float16))
    for lens in ((3000, 17), (4096, 2222)):
        kc, vc = rk.kv4_cache(2, 2, 4096, 64)
        rk.kv4_append(rand(2 * 4096, 2, 64), rand(2 * 4096, 2, 64), kc, vc, torch.zeros(2, dtype=torch.int64, device="cuda"), timed=False)
        q, pos = rand(2, 8, 64), torch.tensor(lens, device="cuda") - 1
        jobs.append((lambda out, q=q, kc=kc, vc=vc, pos=pos: rk.kv4_attn_decode(q, kc, vc, pos, out, timed=False), q.shape, torch.float16))
    for rows in (3, 200):
        x, tok = rand(rows, 5000), torch.arange(rows, device="cuda")
        jobs.append((lambda out, x=x, tok=tok: rk.token_logprobs(x, tok, out, timed=False), (rows,), torch.float32))
    alone = []
    for call, shape, dtype in jobs:
        out = torch.empty(shape, dtype=dtype, device="cuda")
        call(out)
        alone.append(out)
    torch.cuda.synchronize()
    outs = [[[torch.empty(s, dtype=d, device="cuda") for _, s, d in jobs] for _ in range(20)] for _ in range(2)]
    torch.cuda.synchronize()
    failed = []

    def work(mine, order):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for run in mine:
                    for i in order:
                        jobs[i][0](run[i])
                torch.cuda.current_stream().synchronize()
        except Exception as e:                      # handed to the test's own thread
            failed.append(e)
    threads = [threading.Thread(target=work, args=(outs[t], range(len(jobs)) if t == 0 else range(len(jobs) - 1, -1, -1))) for t in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for mine in outs:
        for run in mine:
            for got, want in zip(run, alone):
                assert torch.equal(got, want)


def test_refusals_leave_the_outputs(rk):
    """What the entry points refuse of tensors on the device, with the outputs as they were."""
    z = lambda *shape, dtype=torch.float16: torch.zeros(shape, dtype=dtype, device="cuda")
    q, k, out = z(4, 4, 64), z(4, 2, 64), torch.full((4, 4, 64), 7.0, dtype=torch.float16, device="cuda")
    i32 = lambda *xs: torch.tensor(xs, dtype=torch.int32, device="cuda")
    for call in (lambda: rk.attn_prompt(q, k, k, out[:3]), lambda: rk.attn_prompt(q, k, z(4, 4, 64), out), lambda: rk.attn_prompt(q, z(4, 3, 64), z(4, 3, 64), out),
                 lambda: rk.attn_prompt(q.float(), k, k, out), lambda: rk.attn_prompt(q, k.bfloat16(), k, out), lambda: rk.attn_prompt(z(4, 4, 48), z(4, 2, 48), z(4, 2, 48), z(4, 4, 48)),
                 lambda: rk.attn_prompt(q, k, k, q), lambda: rk.attn_prompt(q, k, k, out, q_start=i32(0)), lambda: rk.attn_prompt(q, k, k, out, k_start=i32(0)),
                 lambda: rk.attn_prompt(q, k, k, out, q_start=i32(0, 4).long()), lambda: rk.attn_prompt(q, z(5, 2, 64), z(5, 2, 64), out, q_start=i32(0, 4)),
                 lambda: rk.attn_prompt(q, k, k, out, lse=z(4, 4)), lambda: rk.attn_prompt(q, k, k, out, scale=0), lambda: rk.attn_prompt(q, k, k, out, max_k=-1),
                 lambda: rk.attn_prompt(q, k, k, out.transpose(1, 2)), lambda: rk.attn_prompt(z(4, 4, 72)[..., 4:68], k, k, out),
                 lambda: rk.attn_prompt(q, k, k, z(1, 4, 64).expand(4, 4, 64)), lambda: rk.attn_prompt(None, k, k, out)):
        with pytest.raises(RuntimeError):
            call()
    kc, vc = rk.kv4_cache(1, 2, 16, 64)
    pos = torch.zeros(1, dtype=torch.int64, device="cuda")
    for call in (lambda: rk.kv4_append(k, k[:2], kc, vc, pos), lambda: rk.kv4_append(k, k, kc, vc, pos.int()), lambda: rk.kv4_append(k, k, kc, kc, pos),
                 lambda: rk.kv4_append(z(4, 3, 64), z(4, 3, 64), kc, vc, pos), lambda: rk.kv4_append(k, k, kc[..., :20], vc[..., :20], pos),
                 lambda: rk.kv4_read(kc, vc, z(17, 2, 64), z(17, 2, 64)), lambda: rk.kv4_read(kc, vc, z(1, 2, 64).expand(4, 2, 64), z(4, 2, 64)),
                 lambda: rk.kv4_attn_decode(z(2, 4, 64), kc, vc, pos, z(2, 4, 64)), lambda: rk.kv4_attn_decode(z(1, 3, 64), kc, vc, pos, z(1, 3, 64)),
                 lambda: rk.kv4_attn_decode(q[:1], kc, vc, pos, out[:1], scale=-1.0), lambda: rk.kv4_attn_decode(q[:1], kc, vc, pos, q[:1]),
                 lambda: rk.kv4_rope_append(z(1, 512), z(15, 32), z(15, 32), pos, z(1, 4, 64), kc, vc), lambda: rk.kv4_rope_append(z(1, 500), z(16, 32), z(16, 32), pos, z(1, 4, 64), kc, vc)):
        with pytest.raises(RuntimeError):
            call()
    x, lp = z(3, 100), torch.full((3,), 7.0, device="cuda")
    tok = torch.zeros(3, dtype=torch.int64, device="cuda")
    for call in (lambda: rk.token_logprobs(x), lambda: rk.token_logprobs(x, None, lp), lambda: rk.token_logprobs(x, tok[:2], lp), lambda: rk.token_logprobs(x, tok.int(), lp),
                 lambda: rk.token_logprobs(x.t(), tok, lp), lambda: rk.token_logprobs(x, tok, z(3)), lambda: rk.token_logprobs(x.double(), tok, lp),
                 lambda: rk.token_logprobs(x, top_ids=z(3, 65, dtype=torch.int64)), lambda: rk.token_logprobs(x, top_ids=z(3, 5, dtype=torch.int64), top_logprobs=z(3, 4, dtype=torch.float32)),
                 lambda: rk.token_logprobs(x, top_ids=z(3, 0, dtype=torch.int64)), lambda: rk.token_logprobs(x.view(1, 3, 100), tok, lp)):
        with pytest.raises(RuntimeError):
            call()
    torch.cuda.synchronize()
    assert bool((out == 7).all()) and bool((lp == 7).all()) and not bool(kc.any()) and not bool(vc.any())
    # empty calls are none
    assert rk.attn_prompt(q[:0], k[:0], k[:0], out[:0]) == 0.0 and rk.token_logprobs(x[:0], tok[:0], lp[:0]) == 0.0
    assert rk.kv4_append(k[:0], k[:0], kc, vc, pos) == 0.0 and rk.kv4_read(kc, vc, k[:0], k[:0]) == 0.0
    # a prompt without keys
    rk.attn_prompt(q, k[:0], k[:0], out, q_start=i32(0, 4), k_start=i32(0), k_len=i32(0))
    assert not bool(out.any())


def test_the_command_scores_packed_windows(rk, capsys):
    """``python -m rptc_kernels.eval_ppl --packed``: the windows and, to the accuracy of two fp16 paths, the loss of the command without it."""
    import json
    args = ["--layers", "1", "--d-model", "256", "--heads", "4", "--d-ff", "704", "--vocab", "500", "--seqlen", "48", "--windows", "5"]
    lines = []
    for extra in ([], ["--packed", "2"]):
        eval_ppl.main(args + extra)
        lines.append(json.loads(capsys.readouterr().out.strip().split("\n")[-1]))
    assert lines[0]["windows"] == lines[1]["windows"] == 5
    assert abs(lines[0]["avg_loss"] - lines[1]["avg_loss"]) < 1e-2 * lines[0]["avg_loss"]
