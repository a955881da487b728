"""The cases by which the attention over whole prompts, the 4-bit key/value cache and the token log probabilities are
timed, with each operator in plain torch operations beside the framework's call.

``own`` False: the plain form (fp32 inside, rounded once at the end).  ``own`` True: the calls a program makes of
``rptc_kernels``."""
import os
import sys

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
GROUP = 32                                  # values of a cache row that share a scale and a minimum


_kernels = None


def _rk():
    global _kernels
    if _kernels is None:
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "let-it-slide_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        import rptc_kernels
        _kernels = rptc_kernels
    return _kernels


# ---------------------------------------------------------------- cases

def listed():
    return [
        # a short chat turn answered by the 32-head model of the decode benchmark: latency is all of it
        {"name": "prompt 37", "op": "prompt", "lens": "37", "past": 0, "heads": 32, "kv_heads": 32, "hd": 128, "dtype": "f16"},
        # the decode benchmark's chunk of 32 tokens at the end of a long context already in the cache: few rows, many keys
        {"name": "chunk 32 after 8000", "op": "prompt", "lens": "32", "past": 8000, "heads": 32, "kv_heads": 32, "hd": 128, "dtype": "f16"},
        # a batch of prompts of very different lengths packed into one call, grouped heads, small head dimension
        {"name": "packed ragged", "op": "prompt", "lens": "1,517,64,2049,0,130,1333", "past": 0, "heads": 16, "kv_heads": 4, "hd": 64, "dtype": "f16"},
        # one long document, grouped heads
        {"name": "prompt 8192", "op": "prompt", "lens": "8192", "past": 0, "heads": 32, "kv_heads": 8, "hd": 128, "dtype": "bf16"},
        # the decode benchmark's prompt of 512 put into a cache of 1024 positions in the middle of a conversation, read back for its attention
        {"name": "store 512 of 1024", "op": "store", "rows": 512, "pos": 411, "batch": 1, "kv_heads": 32, "hd": 128, "max_len": 1024},
        # one new token of each of 7 conversations, small heads
        {"name": "store 7 tokens", "op": "store", "rows": 1, "pos": 300, "batch": 7, "kv_heads": 4, "hd": 64, "max_len": 640},
        # one token of the decode benchmark's loop: prompt 512, the 89th new token
        {"name": "decode 601", "op": "decode", "lens": "601", "heads": 32, "kv_heads": 32, "hd": 128, "max_len": 1024},
        # a serving step: sequences of different lengths, one of them just begun, grouped heads
        {"name": "decode batch 12", "op": "decode", "lens": "1,77,8191,4000,513,2048,6001,333,1024,7777,5000,3333", "heads": 32, "kv_heads": 8, "hd": 128,
         "max_len": 8192},
        # one conversation over a very long document
        {"name": "decode 131072", "op": "decode", "lens": "131007", "heads": 32, "kv_heads": 8, "hd": 128, "max_len": 131072},
        # the token just produced, with the alternatives an interface shows
        {"name": "score 1", "op": "score", "rows": 1, "vocab": 32000, "top": 5, "dtype": "f16"},
        # a perplexity window of 512 predicts 511 tokens; the harness holds fp32 logits
        {"name": "score 511", "op": "score", "rows": 511, "vocab": 32000, "top": 0, "dtype": "f32"},
        # prompt scoring with a large odd vocabulary
        {"name": "score 2048 large", "op": "score", "rows": 2048, "vocab": 128257, "top": 20, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "store", "decode", "decode", "score"])
    if op == "score":
        rows = _log(rng, 1, 2048)
        return {"op": op, "rows": rows, "vocab": _log(rng, 1000, min(128257, 262000000 // rows)), "top": rng.choice([0, 1, 5, 20, 32]),
                "dtype": rng.choice(["f16", "bf16", "f32"])}
    hd = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 8] if kv_heads < 8 else [1, 2, 4])
    if op == "store":
        batch = _log(rng, 1, 8)
        rows, pos = (1, _log(rng, 1, 1000)) if rng.random() < 0.5 else (_log(rng, 2, 1024), rng.randrange(0, 500))
        return {"op": op, "rows": rows, "pos": pos, "batch": batch, "kv_heads": kv_heads, "hd": hd, "max_len": rows + pos + rng.randrange(0, 100)}
    if op == "decode":
        top = _log(rng, 16, 65536)
        lens = [_log(rng, 1, top) for _ in range(_log(rng, 1, 12))]
        return {"op": op, "lens": ",".join(map(str, lens)), "heads": heads, "kv_heads": kv_heads, "hd": hd, "max_len": max(lens) + rng.randrange(0, 64)}
    dtype = rng.choice(["f16", "bf16"])
    if rng.random() < 0.3:
        return {"op": op, "lens": str(_log(rng, 1, 200)), "past": _log(rng, 16, 8000), "heads": heads, "kv_heads": kv_heads, "hd": hd, "dtype": dtype}
    lens = [_log(rng, 1, 2500) for _ in range(rng.randrange(1, 6))]
    return {"op": op, "lens": ",".join(map(str, lens)), "past": 0, "heads": heads, "kv_heads": kv_heads, "hd": hd, "dtype": dtype}


def _lens(case):
    return [int(t) for t in case["lens"].split(",")]


def _row_bytes(hd):
    return hd // 2 + hd // GROUP * 4


def work(case):
    if case["op"] == "score":
        n = case["rows"] * case["vocab"]
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": n * size + case["rows"] * (8 + 8 + 12 * case["top"]), "flops": 5 * n}
    hd, kvh = case["hd"], case["kv_heads"]
    if case["op"] == "store":
        new, back = case["batch"] * case["rows"] * kvh, case["batch"] * (case["pos"] + case["rows"]) * kvh
        # read the new rows, write their records, read every record of the context (the new ones are on chip), write its values
        return {"bytes": 2 * (new * (2 * hd + _row_bytes(hd)) + (back - new) * _row_bytes(hd) + back * 2 * hd), "flops": 2 * (new * 6 * hd + back * 2 * hd)}
    h, lens = case["heads"], _lens(case)
    if case["op"] == "decode":
        return {"bytes": 2 * sum(lens) * kvh * _row_bytes(hd) + 2 * len(lens) * h * hd * 2, "flops": 4 * sum(lens) * h * hd}
    past = case["past"]
    pairs = sum(t * past + t * (t + 1) // 2 for t in lens)
    tq, tk = sum(lens), sum(t + past for t in lens)
    return {"bytes": 2 * hd * (2 * h * tq + 2 * kvh * tk) + 4 * h * tq, "flops": 4 * hd * h * pairs}


# ---------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _channels(g, heads, hd):
    """Spread of a key's channels: a few are several times wider than the others, as in trained models."""
    return 0.6 * torch.exp(0.5 * _randn(g, heads, hd))


def _cache_bytes(g, batch, heads, max_len, hd):
    """Cache rows with every code equally likely, scales and minima as rows of unit spread have them."""
    groups = hd // GROUP
    codes = torch.randint(0, 256, (batch, heads, max_len, hd // 2), generator=g, device="cuda", dtype=torch.uint8)
    scale = 0.27 * torch.exp(0.25 * _randn(g, batch, heads, max_len, groups))
    par = torch.stack([scale, -7.5 * scale * (1 + 0.1 * _randn(g, batch, heads, max_len, groups))], dim=-1).half()
    return torch.cat([codes, par.view(batch, heads, max_len, 2 * groups).view(torch.uint8)], dim=-1).contiguous()


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": dict(case)}
    if case["op"] == "score":
        t, v = case["rows"], case["vocab"]
        # a peaked distribution: a model's logits have a spread of a few units and a handful of likely tokens
        x = 2.5 * _randn(g, t, v)
        x.scatter_add_(1, torch.randint(0, v, (t, 8), generator=g, device="cuda"), 3.0 + 3.0 * torch.rand((t, 8), generator=g, device="cuda"))
        s["logits"] = x.to(DTYPES[case["dtype"]])
        s["tokens"] = torch.randint(0, v, (t,), generator=g, device="cuda")
        return s
    hd, kvh = case["hd"], case["kv_heads"]
    if case["op"] == "store":
        b, t = case["batch"], case["rows"]
        s["k"] = (_randn(g, b * t, kvh, hd) * _channels(g, kvh, hd)).half()
        s["v"] = _randn(g, b * t, kvh, hd).half()
        s["k_cache"] = _cache_bytes(g, b, kvh, case["max_len"], hd)
        s["v_cache"] = _cache_bytes(g, b, kvh, case["max_len"], hd)
        s["pos"] = torch.full((b,), case["pos"], dtype=torch.int64, device="cuda")
        return s
    h, lens = case["heads"], _lens(case)
    if case["op"] == "decode":
        s["q"] = _randn(g, len(lens), h, hd).half()
        s["k_cache"] = _cache_bytes(g, len(lens), kvh, case["max_len"], hd)
        s["v_cache"] = _cache_bytes(g, len(lens), kvh, case["max_len"], hd)
        s["pos"] = torch.tensor(lens, dtype=torch.int64, device="cuda") - 1
        return s
    dt, past, tq = DTYPES[case["dtype"]], case["past"], sum(lens)
    if past:
        # the projection's queries of the chunk, and a cache [kv_heads][positions][hd] with some room behind the context
        s["qkv"] = _randn(g, tq, (h + 2 * kvh) * hd).to(dt)
        s["k_cache"] = (_randn(g, kvh, past + tq + 100, hd) * _channels(g, kvh, hd)[:, None]).to(dt)
        s["v_cache"] = _randn(g, kvh, past + tq + 100, hd).to(dt)
        s["q_start"] = torch.tensor([0, tq], dtype=torch.int32, device="cuda")
        s["k_start"] = torch.zeros(1, dtype=torch.int32, device="cuda")
        s["k_len"] = torch.tensor([past + tq], dtype=torch.int32, device="cuda")
        return s
    # q, k and v side by side, as one projection leaves them
    width = torch.cat([torch.ones(h * hd, device="cuda"), _channels(g, kvh, hd).reshape(-1), torch.ones(kvh * hd, device="cuda")])
    s["qkv"] = (_randn(g, tq, (h + 2 * kvh) * hd) * width).to(dt)
    starts = [0]
    for t in lens:
        starts.append(starts[-1] + t)
    s["q_start"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    s["k_start"] = s["q_start"][:-1].contiguous()
    s["k_len"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    return s


def _qkv(s):
    """q [Tq, heads, hd] and k, v [Tk, kv_heads, hd] of a prompt case, as views."""
    c = s["case"]
    h, kvh, hd = c["heads"], c["kv_heads"], c["hd"]
    q = s["qkv"][:, :h * hd].unflatten(1, (h, hd))
    if c["past"]:
        return q, s["k_cache"].transpose(0, 1), s["v_cache"].transpose(0, 1)
    return q, s["qkv"][:, h * hd:(h + kvh) * hd].unflatten(1, (kvh, hd)), s["qkv"][:, (h + kvh) * hd:].unflatten(1, (kvh, hd))


# ---------------------------------------------------------------- the plain forms

def _plain_prompt(s):
    c = s["case"]
    h, kvh, hd, dt = c["heads"], c["kv_heads"], c["hd"], DTYPES[c["dtype"]]
    q, k, v = _qkv(s)
    tq, tk = q.size(0), k.size(0)
    if c["past"]:
        tk = c["past"] + tq
        k, v = k[:tk], v[:tk]
    rows, cols = torch.arange(tq, device="cuda"), torch.arange(tk, device="cuda")
    # the sequence a query and a key belong to, and the keys in front of the sequence's end
    seq = torch.searchsorted(s["q_start"][1:].long(), rows, right=True)
    first = s["k_start"].long()[seq]
    last = rows - s["q_start"].long()[seq + 1] + s["k_len"].long()[seq] + first
    see = (cols[None, :] >= first[:, None]) & (cols[None, :] <= last[:, None])
    qf = q.float().transpose(0, 1).contiguous()
    kf = k.float().transpose(0, 1).repeat_interleave(h // kvh, dim=0).transpose(1, 2).contiguous()
    vf = v.float().transpose(0, 1).repeat_interleave(h // kvh, dim=0).contiguous()
    x = torch.matmul(qf, kf) * hd ** -0.5
    x = x.masked_fill(~see, float("-inf"))
    m = x.amax(dim=-1, keepdim=True)
    p = torch.exp(x - m)
    l = p.sum(dim=-1, keepdim=True)
    out = torch.matmul(p, vf) / l
    return {"out": out.transpose(0, 1).to(dt).contiguous(), "lse": (m + torch.log(l)).squeeze(-1).t().contiguous()}


def _values(rows, hd):
    """The fp16 values that cache rows [..., bytes] stand for: word w of a row holds dimensions 8w .. 8w+7, its nibble t
    dimension 8w + 2t and its nibble t + 4 dimension 8w + 2t + 1; behind the codes scale and minimum of every group."""
    code = rows[..., :hd // 2].contiguous().view(*rows.shape[:-1], hd // 8, 4)
    nib = torch.stack([code & 15, code >> 4], dim=-1).flatten(-2)                              # [..., word, nibble]
    c = torch.stack([nib[..., :4], nib[..., 4:]], dim=-1).flatten(-2).reshape(*rows.shape[:-1], hd // GROUP, GROUP)
    par = rows[..., hd // 2:].contiguous().view(torch.float16).reshape(*rows.shape[:-1], hd // GROUP, 2).float()
    return (c.float() * par[..., :1] + par[..., 1:]).half().flatten(-2)


def _plain_rows(x):
    """Cache rows of fp16 vectors [..., hd]."""
    hd = x.size(-1)
    g = x.float().unflatten(-1, (hd // GROUP, GROUP))
    lo, hi = g.amin(dim=-1, keepdim=True), g.amax(dim=-1, keepdim=True)
    scale = ((hi - lo) / 15).half()
    sf = scale.float()
    c = torch.where(sf > 0, torch.round((g - lo) / torch.where(sf > 0, sf, 1.0)).clamp(0, 15), 0.0).to(torch.uint8)
    c = c.flatten(-2).unflatten(-1, (hd // 8, 4, 2))
    nib = torch.cat([c[..., 0], c[..., 1]], dim=-1)                                            # [..., word, nibble]
    code = (nib[..., 0::2] | (nib[..., 1::2] << 4)).flatten(-2)
    par = torch.cat([scale, lo.half()], dim=-1).flatten(-2).contiguous().view(torch.uint8)
    return torch.cat([code, par], dim=-1)


def _plain_store(s):
    c = s["case"]
    b, t, kvh, hd = c["batch"], c["rows"], c["kv_heads"], c["hd"]
    n = c["pos"] + t
    for name in ("k", "v"):
        rows = _plain_rows(s[name].unflatten(0, (b, t)).transpose(1, 2))
        s[name + "_cache"][:, :, c["pos"]:n] = rows
    return {name: _values(s[name + "_cache"][:, :, :n], hd).transpose(1, 2).reshape(b * n, kvh, hd).contiguous() for name in ("k", "v")}


def _plain_decode(s):
    c = s["case"]
    h, kvh, hd = c["heads"], c["kv_heads"], c["hd"]
    kf = _values(s["k_cache"], hd).float()                                                     # [n, kv_heads, L, hd]
    vf = _values(s["v_cache"], hd).float()
    q = s["q"].float().unflatten(1, (kvh, h // kvh))
    x = torch.matmul(q, kf.transpose(2, 3).contiguous()) * hd ** -0.5
    see = torch.arange(kf.size(2), device="cuda")[None, :] <= s["pos"][:, None]
    x = x.masked_fill(~see[:, None, None, :], float("-inf"))
    p = torch.exp(x - x.amax(dim=-1, keepdim=True))
    out = torch.matmul(p, vf) / p.sum(dim=-1, keepdim=True)
    return out.flatten(1, 2).half()


def _plain_score(s):
    c = s["case"]
    x = s["logits"].float()
    m = x.amax(dim=-1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    l = e.sum(dim=-1, keepdim=True)
    lse = torch.log(l)
    out = {"logprob": (d.gather(1, s["tokens"][:, None]) - lse).squeeze(1), "entropy": (lse - (d * e).sum(dim=-1, keepdim=True) / l).squeeze(1)}
    if c["top"]:
        # one whole number a logit that orders by value and, for equal values, by the lowest id
        bits = (x + 0.0).view(torch.int32)
        order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
        key = (order << 32) + (0xFFFFFFFF - torch.arange(x.size(1), device="cuda"))
        out["top_ids"] = 0xFFFFFFFF - (torch.topk(key, c["top"], dim=-1).values & 0xFFFFFFFF)
        out["top_logprobs"] = d.gather(1, out["top_ids"]) - lse
    return out


# ---------------------------------------------------------------- one pass

def run(s):
    c = s["case"]
    if not own:
        return {"prompt": _plain_prompt, "store": _plain_store, "decode": _plain_decode, "score": _plain_score}[c["op"]](s)
    rk = _rk()
    if c["op"] == "prompt":
        q, k, v = _qkv(s)
        out = torch.empty((q.size(0), c["heads"], c["hd"]), dtype=q.dtype, device=q.device)
        lse = torch.empty((q.size(0), c["heads"]), dtype=torch.float32, device=q.device)
        rk.attn_prompt(q, k, v, out, q_start=s["q_start"], k_start=s["k_start"], k_len=s["k_len"], lse=lse, timed=False)
        return {"out": out, "lse": lse}
    if c["op"] == "store":
        b, n = c["batch"], c["pos"] + c["rows"]
        rk.kv4_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["pos"], timed=False)
        k = torch.empty((b * n, c["kv_heads"], c["hd"]), dtype=torch.float16, device=s["k"].device)
        v = torch.empty_like(k)
        rk.kv4_read(s["k_cache"], s["v_cache"], k, v, timed=False)
        return {"k": k, "v": v}
    if c["op"] == "decode":
        out = torch.empty_like(s["q"])
        rk.kv4_attn_decode(s["q"], s["k_cache"], s["v_cache"], s["pos"], out, timed=False)
        return out
    t, top = c["rows"], c["top"]
    f32 = {"dtype": torch.float32, "device": s["logits"].device}
    out = {"logprob": torch.empty(t, **f32), "entropy": torch.empty(t, **f32)}
    if top:
        out["top_ids"] = torch.empty((t, top), dtype=torch.int64, device=s["logits"].device)
        out["top_logprobs"] = torch.empty((t, top), **f32)
    rk.token_logprobs(s["logits"], s["tokens"], timed=False, **out)
    return out


# ---------------------------------------------------------------- 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "score":
        x = s["logits"].double()
        logp = x - torch.logsumexp(x, dim=-1, keepdim=True)
        out = {"logprob": logp[torch.arange(x.size(0), device="cuda"), s["tokens"]], "entropy": -(logp.exp() * logp).sum(dim=-1)}
        if case["top"]:
            out["top_ids"] = None
            out["top_logprobs"] = torch.sort(logp, dim=-1, descending=True).values[:, :case["top"]].contiguous() if x.numel() < 30000000 else None
        return out
    hd, kvh = case["hd"], case["kv_heads"]

    def dequantized(rows):
        lead, groups = rows.shape[:-1], hd // GROUP
        par = rows[..., hd // 2:].contiguous().view(torch.float16).double().reshape(*lead, groups, 2)
        out = torch.empty(*lead, hd, dtype=torch.float64, device="cuda")
        for d in range(hd):
            w, t, odd = d // 8, (d % 8) // 2, d % 2
            nibble = t + 4 * odd
            byte = rows[..., 4 * w + nibble // 2]
            code = (byte >> 4 if nibble % 2 else byte & 15).double()
            out[..., d] = code * par[..., d // GROUP, 0] + par[..., d // GROUP, 1]
        return out.half().double()

    if case["op"] == "store":
        b, t, n = case["batch"], case["rows"], case["pos"] + case["rows"]
        res = {}
        for name in ("k", "v"):
            x = s[name].double().reshape(b, t, kvh, hd // GROUP, GROUP)
            lo = x.min(dim=-1, keepdim=True).values
            sc = ((x.max(dim=-1, keepdim=True).values - lo) / 15).half().double()
            code = torch.round((x - lo) / sc.clamp(min=1e-300)).clamp(0, 15) * (sc > 0)
            new = (code * sc + lo).half().double().reshape(b, t, kvh, hd)
            old = dequantized(s[name + "_cache"][:, :, :case["pos"]]).transpose(1, 2)
            res[name] = torch.cat([old, new], dim=1).reshape(b * n, kvh, hd)
        return res
    h, lens = case["heads"], _lens(case)
    if case["op"] == "decode":
        out = torch.empty(len(lens), h, hd, dtype=torch.float64, device="cuda")
        for i, n in enumerate(lens):
            for j in range(kvh):
                kd, vd = dequantized(s["k_cache"][i, j, :n]), dequantized(s["v_cache"][i, j, :n])
                heads = slice(j * (h // kvh), (j + 1) * (h // kvh))
                out[i, heads] = torch.softmax(s["q"][i, heads].double() @ kd.t() / hd ** 0.5, dim=-1) @ vd
        return out
    q, k, v = _qkv(s)
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(q.shape[:2], dtype=torch.float64, device="cuda")
    at = 0
    for n in lens:
        past = case["past"]
        if n == 0:
            continue
        mask = torch.ones(n, past + n, dtype=torch.bool, device="cuda").triu(past + 1)
        for j in range(h):
            g = j // (h // kvh)
            first = 0 if past else at
            x = q[at:at + n, j].double() @ k[first:first + past + n, g].double().t() / hd ** 0.5
            x.masked_fill_(mask, float("-inf"))
            lse[at:at + n, j] = torch.logsumexp(x, dim=-1)
            out[at:at + n, j] = torch.softmax(x, dim=-1) @ v[first:first + past + n, g].double()
        at += n
    return {"out": out, "lse": lse}
