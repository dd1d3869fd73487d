"""The decoder with its KV cache in 8 bits after it has been used: the first
eviction and shift of a large cache, several layers, and set_length to and fro
(test_kv8_model_gpu.py has the new models)."""
import numpy as np
import pytest

import kv8_oracle as O
import neon_cuda as N
import synth as S
from test_kv8_model_gpu import OneLayer, check_moved, close_logits, device, rows_of  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("how", ["evict", "shift"])
def test_first_move_of_a_large_cache(how):
    """The spare cache is made by the call that fills it: 134 MB here, of which a few rows are used."""
    one = OneLayer(ctx=131072, n_head=8, n_kv=8, hd=64)
    for _ in range(3):
        m = N.Model(one.cfg, one.tensors(), kv8=True, kv_weights=True)
        g = np.random.default_rng(5)
        m.forward(g.integers(0, one.cfg.n_vocab, 150))
        before = rows_of(m, 0, 150)
        if how == "shift":
            m.kv_shift(4, 50)
            kept = [np.r_[0:4, 54:150]] * 8
        else:
            m.kv_evict(100, 4, 96)  # no row to choose
            kept = [np.r_[0:4, 54:150]] * 8
        assert m.length == 100
        check_moved(one, m, before, kept, 100)
        tokens = g.integers(0, one.cfg.n_vocab, 3)
        logits = m.forward(tokens)
        close_logits(logits, one.forward(tokens, 100, *rows_of(m, 0, 103))[0])
        m.free()
