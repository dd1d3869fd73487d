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


def gone_over(one, m, tokens, past, valid, step):
    """After set_length(past) on a model with `valid` rows written: they stay, the others are zeros, and so the step runs."""
    before = rows_of(m, 0, valid)
    m.set_length(past)
    k, v = rows_of(m, 0, past)
    for x, y in zip((k, v), before):
        assert np.array_equal(x[:valid], y) and not x[valid:].any()
    logits = m.forward([tokens[step]])
    k, v = rows_of(m, 0, past + 1)
    assert not k[max(valid, past // 32 * 32):past].any() and not v[max(valid, past // 32 * 32):past].any()
    close_logits(logits, one.forward([tokens[step]], past, k, v)[0])


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("steps,to", [(33, 110), (33, 97 + 31), (6, 75), (6, 64 + 6), (1, 159), (0, 90)])
def test_rows_gone_over_in_a_used_model(steps, to, weights):
    """A prompt and single steps fill both slots of the tail; then the length jumps inside the block or across some."""
    one = OneLayer()
    m = N.Model(one.cfg, one.tensors(), kv8=True, kv_weights=weights)
    tokens = np.random.default_rng(6).integers(0, one.cfg.n_vocab, 64 + steps + 1)
    m.forward(tokens[:64])
    for t in tokens[64:64 + steps]:
        m.forward([t])
    gone_over(one, m, tokens, to, 64 + steps, -1)


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("back,to", [(70, 96), (70, 75), (64, 100), (3, 159), (95, 97)])
def test_rows_gone_over_after_a_rewind(back, to, weights):
    """A rewound run's rows do not come back once a step has coded their block anew, nor do their weights."""
    one = OneLayer()
    m = N.Model(one.cfg, one.tensors(), kv8=True, kv_weights=weights)
    tokens = np.random.default_rng(7).integers(0, one.cfg.n_vocab, 102)
    m.forward(tokens[:100])
    m.set_length(back)
    m.forward([tokens[100]])
    gone_over(one, m, tokens, to, back + 1, 101)
    if not weights:
        return
    # of the rows between, those gone over have the last step's weight alone: the rest of them is chosen first
    k, v = rows_of(m, 0, to + 1)
    gone = to - back - 1
    if gone > 1:
        keep = to + 1 - gone
        m.kv_evict(keep, 0, 1)
        assert not any((rows_of(m, 0, keep)[1] == 0).all(axis=(1, 2)))


def test_a_rewind_undone():
    """Without a step between, set_length brings the rows back, and their tail: the cache is as if it had not been called."""
    one = OneLayer()
    a, b = (N.Model(one.cfg, one.tensors(), kv8=True) for _ in range(2))
    tokens = np.random.default_rng(8).integers(0, one.cfg.n_vocab, 90)
    for m in (a, b):
        m.forward(tokens[:75])
    a.set_length(10)
    a.set_length(50)
    a.set_length(75)
    for m in (a, b):
        m.forward(tokens[75:])
    for x, y in zip(rows_of(a, 0, 90), rows_of(b, 0, 90)):
        assert np.array_equal(x, y)


def test_rows_gone_over_after_an_eviction():
    one = OneLayer()
    m = N.Model(one.cfg, one.tensors(), kv8=True, kv_weights=True)
    tokens = np.random.default_rng(9).integers(0, one.cfg.n_vocab, 121)
    m.forward(tokens[:120])
    m.kv_evict(41, 4, 20)
    gone_over(one, m, tokens, 100, 41, -1)
    m.set_length(90)
    m.kv_shift(2, 30)  # 60 rows
    gone_over(one, m, tokens, 119, 60, -1)


def test_memory_beyond_the_cache():
    """A model with an 8-bit cache of 131072 rows holds the cache, the RoPE table and a few MB, and no room for the
    weights that it does not keep; reading rows takes no buffer of the cache's length."""
    one = OneLayer(ctx=131072, n_embd=128, n_head=8, n_kv=8, hd=128)
    cache, table = 2 * 8 * 131072 * (128 + 4 / 32), 131072 * 64 * 8
    torch.cuda.synchronize()

    def used():
        return torch.cuda.mem_get_info()[1] - torch.cuda.mem_get_info()[0]

    N.Model(one.cfg, one.tensors(), kv8=True).free()  # the library's own set-up
    start = used()
    m = N.Model(one.cfg, one.tensors(), kv8=True)
    tokens = np.random.default_rng(10).integers(0, one.cfg.n_vocab, 9000)
    m.forward(tokens[:300])
    assert used() - start <= cache + table + (48 << 20)
    for t in range(300, 9000, 900):
        m.forward(tokens[t:t + 900])
    n = m.length
    k, v = rows_of(m, 0, n)  # in pieces
    k1, v1 = rows_of(m, 0, 40)
    assert np.array_equal(k[:40], k1) and np.array_equal(v[:40], v1) and (np.abs(k).max(axis=(1, 2)) > 0).all()
    assert used() - start <= cache + table + (72 << 20)
    m.kv_shift(4, 100)
    assert used() - start <= 2 * cache + table + (84 << 20)
    k2, v2 = rows_of(m, 0, n - 100)
    half = n // 2 // 32 * 32
    assert np.abs(v2[half:half + 32] - v[half + 100:half + 132]).max() <= np.abs(v[half + 100:half + 132]).max() / 100
    m.free()


def test_layers_do_not_mix():
    """Three layers share one spare cache: each keeps rows of its own, twice over."""
    cfg = S.ModelConfig(300, 128, 3, 4, 2, 64, 128, ctx_len=256, rope_base=1e4)
    m = N.Model(cfg, list(S.model_tensors(cfg, seed=5)), kv8=True, kv_weights=True)
    g = np.random.default_rng(11)
    m.forward(g.permutation(cfg.n_vocab)[:200])  # (rows of the same token are the same in layer 0)
    for keep, sink, recent in ((120, 4, 30), (61, 2, 20)):
        n = m.length
        before = [rows_of(m, li, n) for li in range(3)]
        m.kv_evict(keep, sink, recent)
        chosen = []
        for li in range(3):
            v = rows_of(m, li, keep)[1]
            for h in range(cfg.n_kv_head):
                old = before[li][1][:, h]
                r = np.array([np.abs(old - x).max(1).argmin() for x in v[:, h]])
                step = np.repeat([np.abs(v[b:b + 32, h]).max() / 127 for b in range(0, keep, 32)], 32)[:keep]
                assert (np.abs(old[r] - v[:, h]).max(1) <= step * (0.5 + 2.0 ** -10)).all()  # a row of this layer, coded again
                assert (np.diff(r) > 0).all() and np.array_equal(r[:sink], np.arange(sink))
                assert np.array_equal(r[keep - recent:], np.arange(n - recent, n))
                chosen.append(tuple(r))
        assert len(set(chosen)) > 1  # by each head's own weights
        before = [rows_of(m, li, keep) for li in range(3)]
        m.kv_shift(1, 5)
        for li in range(3):
            v = rows_of(m, li, keep - 5)[1]
            want = np.concatenate([before[li][1][:1], before[li][1][6:]])
            for h in range(cfg.n_kv_head):
                assert np.array_equal(v[:, h], O.values(*O.quantise(want[:, h])))
        m.forward(g.integers(0, cfg.n_vocab, 9))


def test_an_eviction_without_memory_can_be_tried_again():
    """Too little memory for the spare cache is an error that costs nothing: not the rows, and no memory per attempt."""
    one = OneLayer(ctx=131072, n_head=8, n_kv=8, hd=128, n_embd=128)
    m = N.Model(one.cfg, one.tensors(), kv8=True, kv_weights=True)
    tokens = np.random.default_rng(12).integers(0, one.cfg.n_vocab, 103)
    m.forward(tokens[:100])
    before = rows_of(m, 0, 100)
    torch.cuda.empty_cache()
    hold = []
    while torch.cuda.mem_get_info()[0] > 200 << 20:  # the spare cache takes 269 MB
        hold.append(torch.empty(max(2 << 20, torch.cuda.mem_get_info()[0] - (160 << 20)), dtype=torch.uint8, device="cuda"))
    used = []
    for _ in range(4):
        with pytest.raises(RuntimeError, match="cudaMalloc"):
            m.kv_evict(50, 4, 46)
        used.append(torch.cuda.mem_get_info()[0])
        torch.cuda.synchronize()
    assert len(set(used)) == 1
    assert m.length == 100 and all(np.array_equal(a, b) for a, b in zip(rows_of(m, 0, 100), before))
    m.forward(tokens[100:])  # (nor is it the next step's error)
    m.set_length(100)
    before = rows_of(m, 0, 100)  # (the step coded the last block anew)
    del hold
    torch.cuda.empty_cache()
    m.kv_evict(50, 4, 46)
    check_moved(one, m, before, [np.r_[0:4, 54:100]] * 8, 50)
