"""What QuantizedLlama refuses before it runs anything (no device is touched)."""
from types import SimpleNamespace

import pytest
import torch

from rptc_kernels import eval_ppl
from rptc_kernels.llama_decode import LlamaShape, QuantizedLlama

SHAPE = LlamaShape(layers=1, d_model=64, heads=1, d_ff=64, vocab=10, max_len=40)


def model(**kw):
    def layers(*args):
        raise AssertionError("the layers ran")
    return SimpleNamespace(shape=SHAPE, embed=torch.zeros(10, 64), _layers=layers, **kw)


@pytest.mark.parametrize("tokens", [[0, 3, 10], [-1, 2], [1 << 40], [9, 9, 9, -(1 << 40)]])
def test_tokens_outside_the_vocabulary(tokens):
    # on a device such an index ends the process
    m = model(cache_bits=16)
    m.forward_prompt = lambda *a, **kw: QuantizedLlama.forward_prompt(m, *a, **kw)
    with pytest.raises(ValueError, match="vocabulary"):
        m.forward_prompt(torch.tensor(tokens))
    with pytest.raises(ValueError, match="vocabulary"):
        eval_ppl.score_tokens(m, tokens)


@pytest.mark.parametrize("pos", [[0, 2], [5, 4], [3, 3], [-1, 0], [39, 40], [0, 1, 2, 7]])
def test_a_chunk_on_a_4_bit_cache_whose_positions_do_not_follow_each_other(pos):
    # its rows are appended one behind the other from the first position on, and its last query sees all up to its own
    m = model(cache_bits=4, _attend_kv4=None)
    with pytest.raises(ValueError, match="position"):
        QuantizedLlama.forward_tokens(m, torch.zeros(len(pos), dtype=torch.int64), torch.tensor(pos))
    with pytest.raises(AssertionError, match="the layers ran"):
        QuantizedLlama.forward_tokens(m, torch.zeros(3, dtype=torch.int64), torch.tensor([37, 38, 39]))
