"""generate()'s options that do not go together are refused before anything runs."""
import pytest
import torch

import generate as G
from midiemo.vocab import get_maps


class Untouched:
    """a model of which generate() may ask no forward"""
    vocab_size = 1007

    def to(self, device):
        return self

    def eval(self):
        return self


@pytest.mark.parametrize("kv_bits", [4, 8])
def test_a_quantised_cache_needs_a_cache(kv_bits):
    call = lambda **kw: G.generate(Untouched(), get_maps(n_emotion_bins=0), torch.device("cpu"), "/tmp/none", "continuous_concat", gen_len=4, debug=True, kv_bits=kv_bits, **kw)
    with pytest.raises(ValueError, match="kv_bits"):
        call(continuous_conditions=[[0.0, 0.0]], use_cache=False)
    with pytest.raises(ValueError, match="kv_bits"):                # a condition that changes from step to step recomputes every position: no cache either
        call(varying_condition=[torch.zeros(1, 4), torch.zeros(1, 4)])
