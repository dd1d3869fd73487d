"""The decoder with its KV cache in 8 bits (neon_cuda_model_create_kv8): the
cache against the fp32 model's, logits against float64 over the cached values,
generation, the window's shift, and eviction by accumulated weight.

Logits: a one-layer model of F32 weights whose ffn_down is zero is a chain of
four fp32 products (256 terms at most: 2^-16 of the sum of magnitudes each),
the attention (test_kv8_gpu.py) and two norms, against float64; 2^-11 of the
largest logit bounds it with the chain's growth (the products' sums of
magnitudes are at most 16 times the results' size here)."""
import numpy as np
import pytest

import kv8_oracle as O
import neon_cuda as N
import synth as S

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
TINY = S.ModelConfig(1000, 256, 2, 4, 2, 64, 512, ctx_len=64, rope_base=1e4, name="tiny")


@pytest.fixture(scope="module", autouse=True)
def device():
    assert torch.cuda.is_available()
    N.init(0)


class OneLayer:
    """A one-layer decoder of F32 weights without an FFN, and its forward pass in float64."""

    def __init__(self, ctx=160, n_vocab=300, n_embd=128, n_head=6, n_kv=2, hd=64, rope_dim=0, seed=1):
        self.cfg = S.ModelConfig(n_vocab, n_embd, 1, n_head, n_kv, hd, 64, ctx_len=ctx, rope_base=1e4,
                                 rope_dim_count=rope_dim)
        g = np.random.default_rng(seed)
        w = lambda *s: (g.standard_normal(s) / np.sqrt(s[-1])).astype(np.float32)  # noqa: E731
        q, kv = n_head * hd, n_kv * hd
        self.t = {0: w(n_vocab, n_embd) * 4, 1: np.ones((1, n_embd), np.float32), 2: w(n_vocab, n_embd),
                  3: np.ones((1, n_embd), np.float32), 4: w(q, n_embd) * 2, 5: w(kv, n_embd), 6: w(kv, n_embd),
                  7: w(n_embd, q), 8: np.ones((1, n_embd), np.float32), 9: w(64, n_embd), 10: w(64, n_embd),
                  11: np.zeros((n_embd, 64), np.float32)}

    def tensors(self):
        for role, a in self.t.items():
            norm = role in (1, 3, 8)
            yield (role, 0 if role >= 3 else -1, a.reshape(-1).view(np.uint8), N.GGML_F32, a.shape[1],
                   0 if norm else a.shape[0])

    def norm(self, x):
        return x / np.sqrt(np.mean(x * x, -1, keepdims=True) + self.cfg.norm_eps)

    def rotate(self, x, pos):
        """x [n, heads, hd]: pairs (2i, 2i + 1)."""
        hd = self.cfg.head_dim
        half = (self.cfg.rope_dim_count or hd) // 2
        a = pos[:, None] / self.cfg.rope_scale * self.cfg.rope_base ** (-2.0 * np.arange(half) / hd)
        c, s = np.cos(a)[:, None], np.sin(a)[:, None]
        y = x.copy()
        p, q = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = p * c - q * s, p * s + q * c
        return y

    def forward(self, tokens, past, k, v):
        """Logits of the last token and the weight of each row, over cached values k, v [rows, H, hd]."""
        c, t = self.cfg, {r: a.astype(np.float64) for r, a in self.t.items()}
        h = t[0][tokens]
        x = self.norm(h)
        q = self.rotate((x @ t[4].T).reshape(len(tokens), c.n_head, c.head_dim), past + np.arange(len(tokens)))
        o, w, _ = O.attention(q, k.transpose(1, 0, 2), v.transpose(1, 0, 2), past, c.head_dim ** -0.5)
        h = h + o.reshape(len(tokens), -1) @ t[7].T
        return t[2] @ self.norm(h[-1]), w


def rows_of(m, layer, n):
    c = m.cfg
    k, v = m.read_kv(layer, n)
    return k.reshape(n, c.n_kv_head, c.head_dim), v.reshape(n, c.n_kv_head, c.head_dim)


def close_logits(got, want):
    assert np.abs(got - want).max() <= 2.0 ** -11 * np.abs(want).max()


def test_first_layer_is_the_float_models_in_8_bits():
    """Layer 0's K and V do not depend on the attention: the codes are those of the fp32 model's rows."""
    tensors = list(S.model_tensors(TINY, seed=3))
    prompt = S.prompt_tokens(41, TINY.n_vocab, 4)
    f, e = N.Model(TINY, tensors), N.Model(TINY, tensors, kv8=True)
    for m in (f, e):
        m.forward(prompt)
        for t in (5, 6, 7, 8):
            m.forward([t])
    n = 45
    for a, b in zip(rows_of(f, 0, n), rows_of(e, 0, n)):
        for h in range(TINY.n_kv_head):
            assert np.array_equal(O.values(*O.quantise(a[:, h])), b[:, h])


@pytest.mark.parametrize("kw", [dict(), dict(hd=128, n_head=4, n_kv=1), dict(rope_dim=32), dict(hd=96, n_head=2, n_kv=2)])
def test_logits_over_the_cached_values(kw):
    one = OneLayer(**kw)
    m = N.Model(one.cfg, one.tensors(), kv8=True)
    g = np.random.default_rng(2)
    past = 0
    for n in (70, 1, 1, 5, 1, 40):
        tokens = g.integers(0, one.cfg.n_vocab, n)
        logits = m.forward(tokens)
        k, v = rows_of(m, 0, past + n)
        close_logits(logits, one.forward(tokens, past, k, v)[0])
        past += n
    m.set_length(75)  # rewound, and on
    tokens = g.integers(0, one.cfg.n_vocab, 3)
    logits = m.forward(tokens)
    close_logits(logits, one.forward(tokens, 75, *rows_of(m, 0, 78))[0])


@pytest.mark.parametrize("start", [5, 32, 45, 159])
def test_rows_gone_over_are_zeros(start):
    """set_length beyond what was written: those rows are zeros, as in the fp32 cache, and have no weight yet."""
    one = OneLayer()
    m = N.Model(one.cfg, one.tensors(), kv8=True, kv_weights=True)
    m.set_length(start)
    out = m.forward([7])
    k, v = rows_of(m, 0, start + 1)
    assert not k[:start].any() and not v[:start].any()
    want, _ = one.forward([7], start, k, v)
    close_logits(out, want)
    if start > 8:
        m.kv_evict(8, 2, 2)
        k, v = rows_of(m, 0, 8)
        assert not k[:7].any() and k[7].any()


def test_generate_is_forward_step_by_step():
    tensors = list(S.model_tensors(TINY, seed=3))
    prompt = S.prompt_tokens(12, TINY.n_vocab, 4)
    a, b = N.Model(TINY, tensors, kv8=True, kv_weights=True), N.Model(TINY, tensors, kv8=True)
    toks = a.generate(prompt, 20)  # the graph
    logits = b.forward(prompt)
    for t in toks:
        assert int(np.argmax(logits)) == t
        logits = b.forward([t])
    assert a.length == b.length == 32
    for layer in range(TINY.n_layer):
        for x, y in zip(rows_of(a, layer, 31), rows_of(b, layer, 31)):
            assert np.array_equal(x, y)


def test_two_models_take_turns():
    tensors = list(S.model_tensors(TINY, seed=3))
    p, q = S.prompt_tokens(10, TINY.n_vocab, 4), S.prompt_tokens(15, TINY.n_vocab, 5)
    alone = [N.Model(TINY, tensors, kv8=True).generate(x, 8) for x in (p, q)]
    a, b = N.Model(TINY, tensors, kv8=True), N.Model(TINY, tensors, kv8=True)
    assert np.array_equal(a.generate(p, 4), alone[0][:4]) and np.array_equal(b.generate(q, 8), alone[1])
    assert np.array_equal(a.generate(alone[0][3:4], 4), alone[0][4:])


def check_moved(one, m, before, kept, n):
    """The cache's rows are the kept ones of `before` (k, v as values), K rotated."""
    k, v = rows_of(m, 0, n)
    for h in range(one.cfg.n_kv_head):
        r = np.asarray(kept[h])
        same = np.repeat([(r[b:b + 32] == np.arange(b, b + len(r[b:b + 32]))).all() for b in range(0, n, 32)], 32)[:n]
        want = np.where(same[:, None], before[1][r, h], O.values(*O.quantise(before[1][r, h])))
        assert np.array_equal(v[:, h], want)
        x = one.rotate(before[0][r][:, h:h + 1].astype(np.float64), (np.arange(n) - r).astype(np.float64))[:, 0]
        # a code's step of the new block, half of it by rounding, and fp32 angles
        step = np.repeat([np.abs(x[b:b + 32]).max() / 127 for b in range(0, n, 32)], 32)[:n]
        assert (np.abs(k[:, h] - x) <= step[:, None] * (0.5 + 2.0 ** -9)).all()


def test_shift():
    one = OneLayer(rope_dim=48)
    m = N.Model(one.cfg, one.tensors(), kv8=True, kv_weights=True)
    g = np.random.default_rng(3)
    m.forward(g.integers(0, one.cfg.n_vocab, 150))
    before = rows_of(m, 0, 150)
    m.kv_shift(4, 50)
    assert m.length == 100
    kept = np.r_[0:4, 54:150]
    check_moved(one, m, before, [kept] * 2, 100)
    m.kv_shift(100, 5)  # nothing to slide
    m.kv_shift(0, 0)
    assert m.length == 100
    tokens = g.integers(0, one.cfg.n_vocab, 7)
    logits = m.forward(tokens)
    close_logits(logits, one.forward(tokens, 100, *rows_of(m, 0, 107))[0])


def test_evict():
    """The rows that stay are those of the largest weight, summed over all queries so far in float64."""
    one = OneLayer()
    m = N.Model(one.cfg, one.tensors(), kv8=True, kv_weights=True)
    g = np.random.default_rng(4)
    past, weight = 0, np.zeros((2, 0))
    for n in (90, 1, 1, 4, 1, 30, 1):
        tokens = g.integers(0, one.cfg.n_vocab, n)
        m.forward(tokens)
        _, w = one.forward(tokens, past, *rows_of(m, 0, past + n))
        weight = np.concatenate([weight, np.zeros((2, n))], 1) + w
        past += n
    m.kv_evict(past, 4, 4)  # holds no more
    assert m.length == past
    keep, sink, recent = 70, 4, 20
    before = rows_of(m, 0, past)
    kept = [O.evicted(weight[h], past, keep, sink, recent) for h in range(2)]
    for h in range(2):  # the choice is clear of fp32's rounding
        mid = np.sort(weight[h, sink:past - recent])[::-1]
        cut = keep - sink - recent
        assert mid[cut - 1] - mid[cut] > 1e-5 * mid[cut]
    m.kv_evict(keep, sink, recent)
    assert m.length == keep
    check_moved(one, m, before, kept, keep)
    tokens = g.integers(0, one.cfg.n_vocab, 5)
    logits = m.forward(tokens)
    close_logits(logits, one.forward(tokens, keep, *rows_of(m, 0, keep + 5))[0])
    assert len(m.generate(tokens, 30)) == 30  # the window goes on
    m.kv_evict(40, 0, 40)
    assert m.length == 40


def test_refusals():
    tensors = list(S.model_tensors(TINY, seed=3))
    m = N.Model(TINY, tensors, kv8=True)
    m.forward([1, 2, 3])
    with pytest.raises(RuntimeError, match="does not keep attention weights"):
        m.kv_evict(2, 0, 0)
    with pytest.raises(RuntimeError, match="kv_weights needs kv8"):
        N.Model(TINY, tensors, kv_weights=True)
    w = N.Model(TINY, tensors, kv8=True, kv_weights=True)
    for bad in ((0, 0, 0), (TINY.ctx_len + 1, 0, 0), (4, 5, 0), (4, 2, 3)):
        with pytest.raises(RuntimeError, match="kv_evict"):
            w.kv_evict(*bad)
    with pytest.raises(RuntimeError, match="KV cache exhausted"):
        m.forward(np.zeros(TINY.ctx_len, np.int32))
    far = S.ModelConfig(64, 32, 1, 1, 1, 32, 32, ctx_len=20000, rope_base=1e4)
    with pytest.raises(RuntimeError, match="16384"):
        N.Model(far)
    N.Model(far, kv8=True).free()
    with pytest.raises(RuntimeError, match="131072"):
        N.Model(S.ModelConfig(64, 32, 1, 1, 1, 32, 32, ctx_len=131073, rope_base=1e4), kv8=True)
