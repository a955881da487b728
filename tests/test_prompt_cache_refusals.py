"""Calls of the prompt attention, the 4-bit cache and the token log probabilities that are refused, or are not, before a device is
touched: by the C ABI's statuses (no pointer here is ever read)."""
import ctypes

import pytest
import torch

import rptc_kernels as rk

ESHAPE, EALIAS = -2, -7
REFUSED = (-1, -2, -3, -4, -5, -7)              # every status of the checks in front of the device's


@pytest.fixture(scope="module")
def lib():
    return rk.library()


def logprobs(lib, logits=1 << 16, tokens=1 << 30, logprob=None, entropy=None, ids=None, tops=None, rows=4, vocab=1000, top=0):
    return lib.rptc_token_logprobs(logits, 0, tokens, logprob, entropy, ids, tops, rows, vocab, vocab, top, None, None)


def test_scores_over_the_tokens_or_over_each_other(lib):
    t, a = 1 << 30, 1 << 31
    assert logprobs(lib, tokens=t, logprob=t) == EALIAS and logprobs(lib, tokens=t, logprob=t + 28) == EALIAS
    assert logprobs(lib, tokens=t, logprob=a, entropy=t - 12) == EALIAS and logprobs(lib, tokens=t, ids=t, top=1) == EALIAS
    assert logprobs(lib, logprob=a, entropy=a) == EALIAS and logprobs(lib, logprob=a, entropy=a + 12) == EALIAS
    assert logprobs(lib, logprob=a, ids=a - 8 * 4 * 3 + 4, top=3) == EALIAS and logprobs(lib, entropy=a, tops=a + 15, top=2) == EALIAS
    assert logprobs(lib, ids=a, tops=a + 8 * 4 * 2 - 4, top=2) == EALIAS
    # side by side they are not
    for call in (dict(tokens=t, logprob=t + 32), dict(tokens=t, logprob=t - 16), dict(logprob=a, entropy=a + 16), dict(ids=a, tops=a + 64, top=2)):
        if not torch.cuda.is_available():
            assert logprobs(lib, **call) not in (0,) + REFUSED


def test_rows_read_back_over_each_other(lib):
    kc, vc, k, v = 1 << 22, 1 << 23, 1 << 20, 1 << 21

    def read(seqs=1, rows=4, kv_heads=2, st=(128, 64, 128, 64)):
        return lib.rptc_kv4_read(kc, vc, k, v, seqs, rows, kv_heads, 64, 16, *st, None, None)
    for i in range(4):
        st = [128, 64, 128, 64]
        st[i] = 0
        assert read(st=st) == ESHAPE
        if not torch.cuda.is_available():       # one row, one head: its stride means nothing
            assert read(rows=1, kv_heads=1, st=st) not in (0,) + REFUSED
    assert read(seqs=2, rows=1, st=(0, 64, 128, 64)) == ESHAPE


@pytest.mark.skipif(torch.cuda.is_available(), reason="with a device the call would read its pointers")
def test_one_query_for_all_rows_or_heads_is_not_refused(lib):
    # strides of 0 repeat what is read; what is written may not repeat
    for st, refused in (((0, 64, 128, 64, 128, 64, 256, 64), False), ((256, 0, 128, 64, 128, 64, 256, 64), False), ((0, 0, 0, 0, 0, 0, 256, 64), False),
                        ((256, 64, 128, 64, 128, 64, 0, 64), True), ((256, 64, 128, 64, 128, 64, 256, 0), True)):
        rc = lib.rptc_attn_prompt(16, 1 << 20, 1 << 21, 1 << 22, None, None, None, None, 1, 8, 8, 8, 4, 2, 64, ctypes.byref(rk.PromptStrides(*st)),
                                  0.125, 1, 0, None, 0, None, None)
        assert (rc == ESHAPE) if refused else rc not in (0,) + REFUSED
