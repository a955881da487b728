"""What the prompt attention, the 4-bit cache and the token log probabilities refuse before they touch a device: the C ABI by
its statuses (no pointer here is ever read), the Python functions by their errors."""
import ctypes

import pytest
import torch

import rptc_kernels as rk

ENULL, ESHAPE, EALIGN, EMODE, ELIMIT, EALIAS = -1, -2, -3, -4, -5, -7


@pytest.fixture(scope="module")
def lib():
    return rk.library()


def prompt(lib, *, q=16, k=1 << 20, v=1 << 21, out=1 << 22, lse=None, q_start=None, k_start=None, k_len=None, seqs=1, total_q=8,
           total_k=8, max_k=8, heads=4, kv_heads=2, hd=64, strides="contiguous", scale=0.125, causal=1, dtype=0, workspace=None, size=0):
    if strides == "contiguous":
        strides = (heads * hd, hd, kv_heads * hd, hd, kv_heads * hd, hd, heads * hd, hd)
    if strides is not None:
        strides = ctypes.byref(rk.PromptStrides(*strides))
    return lib.rptc_attn_prompt(q, k, v, out, lse, q_start, k_start, k_len, seqs, total_q, total_k, max_k, heads, kv_heads, hd, strides,
                                scale, causal, dtype, workspace, size, None, None)


@pytest.mark.parametrize("bad, status", [
    (dict(q=None), ENULL), (dict(out=None), ENULL), (dict(strides=None), ENULL),
    (dict(q=8), EALIGN), (dict(k=(1 << 20) + 2), EALIGN), (dict(strides=(260, 64, 128, 64, 128, 64, 256, 64)), EALIGN),
    (dict(hd=48), ESHAPE), (dict(hd=512), ESHAPE), (dict(heads=5), ESHAPE), (dict(kv_heads=0), ESHAPE), (dict(total_q=-1), ESHAPE),
    (dict(max_k=-1), ESHAPE), (dict(dtype=2), EMODE), (dict(dtype=-1), EMODE), (dict(scale=0.0), ESHAPE),
    (dict(scale=float("nan")), ESHAPE), (dict(scale=float("inf")), ESHAPE), (dict(seqs=2), ESHAPE), (dict(k_start=16), ENULL),
    (dict(total_q=(1 << 24) + 1), ELIMIT), (dict(heads=2048, kv_heads=2048), ELIMIT),
    (dict(k=1 << 22), EALIAS), (dict(out=16), EALIAS),
])
def test_prompt_statuses(lib, bad, status):
    assert prompt(lib, **bad) == status


def test_kv4_statuses(lib):
    assert [lib.rptc_kv4_row_bytes(hd) for hd in (32, 64, 128, 256, 48, 0, -32)] == [20, 40, 80, 160, ESHAPE, ESHAPE, ESHAPE]
    k, v, kc, vc, pos = 1 << 20, 1 << 21, 1 << 22, 1 << 23, 1 << 24

    def append(k=k, v=v, kc=kc, vc=vc, pos=pos, q_start=None, seqs=1, total=4, kv_heads=2, hd=64, max_len=16, st=(128, 64, 128, 64)):
        return lib.rptc_kv4_append(k, v, kc, vc, pos, q_start, seqs, total, kv_heads, hd, max_len, *st, None, None)
    assert append(k=None) == ENULL and append(pos=None) == ENULL
    assert append(hd=48) == ESHAPE and append(seqs=0) == ESHAPE and append(total=5, seqs=2) == ESHAPE and append(max_len=0) == ESHAPE
    assert append(k=k + 2) == EALIGN and append(st=(132, 64, 128, 64)) == EALIGN
    assert append(seqs=65536, total=65536) == ELIMIT and append(max_len=(1 << 26) + 1) == ELIMIT
    assert append(kc=k) == EALIAS and append(vc=kc) == EALIAS

    def read(k=k, v=v, kc=kc, vc=vc, seqs=1, rows=4, kv_heads=2, hd=64, max_len=16, st=(128, 64, 128, 64)):
        return lib.rptc_kv4_read(kc, vc, k, v, seqs, rows, kv_heads, hd, max_len, *st, None, None)
    assert read(v=None) == ENULL and read(hd=16) == ESHAPE and read(rows=17) == ESHAPE and read(rows=-1) == ESHAPE
    assert read(v=v + 8) == EALIGN and read(k=kc) == EALIAS and read(v=k) == EALIAS

    def rope(qkv=16, cos=1 << 16, sin=1 << 17, pos=pos, q=k, kc=kc, vc=vc, seqs=1, heads=4, kv_heads=2, hd=64, max_len=16):
        return lib.rptc_kv4_rope_append(qkv, cos, sin, pos, q, kc, vc, seqs, heads, kv_heads, hd, max_len, None, None)
    assert rope(cos=None) == ENULL and rope(heads=3) == ESHAPE and rope(hd=512) == ESHAPE and rope(qkv=18) == EALIGN
    assert rope(q=16) == EALIAS and rope(heads=2048, kv_heads=2048) == ELIMIT

    def decode(q=16, kc=kc, vc=vc, pos=pos, out=1 << 30, seqs=1, heads=4, kv_heads=2, hd=64, max_len=16, q_token=256, ws=None, size=0):
        return lib.rptc_kv4_attn_decode(q, kc, vc, pos, out, seqs, heads, kv_heads, hd, max_len, q_token, 0.125, ws, size, None, None)
    assert decode(out=None) == ENULL and decode(heads=3) == ESHAPE and decode(hd=96) == ESHAPE and decode(q_token=260) == EALIGN
    assert decode(out=16) == EALIAS and decode(heads=1026, kv_heads=2) == ELIMIT


def test_logprob_statuses(lib):
    def call(logits=16, dtype=0, tokens=1 << 30, logprob=1 << 31, entropy=None, ids=None, tops=None, rows=4, vocab=1000, stride=1000, top=0):
        return lib.rptc_token_logprobs(logits, dtype, tokens, logprob, entropy, ids, tops, rows, vocab, stride, top, None, None)
    assert call(logits=None) == ENULL and call(tokens=None) == ENULL and call(logprob=None) == ENULL and call(top=3) == ESHAPE
    assert call(dtype=3) == EMODE and call(vocab=0) == ESHAPE and call(stride=-1) == ESHAPE and call(rows=-1) == ESHAPE
    assert call(top=-1) == ESHAPE and call(top=65, ids=1 << 32, tops=1 << 33) == ELIMIT and call(top=9, vocab=8, ids=1 << 32) == ESHAPE
    assert call(rows=1 << 22) == ELIMIT and call(vocab=1 << 30, stride=1 << 30) == ELIMIT and call(logits=17) == EALIGN
    assert call(logits=1 << 16, logprob=(1 << 16) + 4 * 1000) == EALIAS and call(logits=1 << 16, entropy=(1 << 16) - 4) == EALIAS


@pytest.mark.parametrize("call", [
    lambda h: rk.attn_prompt(h(4, 4, 64), h(4, 2, 64), h(4, 2, 64), h(4, 4, 64)),
    lambda h: rk.kv4_append(h(4, 2, 64), h(4, 2, 64), *rk.kv4_cache(1, 2, 16, 64, device="cpu"), torch.zeros(1, dtype=torch.int64)),
    lambda h: rk.kv4_read(*rk.kv4_cache(1, 2, 16, 64, device="cpu"), h(4, 2, 64), h(4, 2, 64)),
    lambda h: rk.kv4_rope_append(h(1, 512), h(16, 32), h(16, 32), torch.zeros(1, dtype=torch.int64), h(1, 4, 64),
                                 *rk.kv4_cache(1, 2, 16, 64, device="cpu")),
    lambda h: rk.kv4_attn_decode(h(1, 4, 64), *rk.kv4_cache(1, 2, 16, 64, device="cpu"), torch.zeros(1, dtype=torch.int64), h(1, 4, 64)),
    lambda h: rk.token_logprobs(h(4, 100), torch.zeros(4, dtype=torch.int64), torch.zeros(4)),
])
def test_cpu_tensors_are_rejected_not_computed(call):
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        call(lambda *shape: torch.zeros(shape, dtype=torch.float16))


def test_cache_sizes_and_model_arguments():
    kc, vc = rk.kv4_cache(3, 2, 10, 128, device="cpu")
    assert kc.shape == vc.shape == (3, 2, 10, 80) and kc.dtype == torch.uint8 and not kc.any()
    with pytest.raises((RuntimeError, ValueError)):
        rk.kv4_cache(1, 1, 8, 48, device="cpu")
    from rptc_kernels.llama_decode import LlamaShape, QuantizedLlama
    with pytest.raises(ValueError):
        QuantizedLlama(LlamaShape(layers=1, d_model=64, heads=1, d_ff=64, vocab=8, max_len=8), device="cpu", cache_bits=8)
    from rptc_kernels import eval_ppl
    for args in ((torch.arange(3), 8), (torch.arange(8), 1), (torch.arange(8), 4, 0)):
        with pytest.raises(ValueError):
            eval_ppl.packed_perplexity(None, *args)
