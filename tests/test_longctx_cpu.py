"""The long-context operators' argument checks, on a host without a GPU: each
refusal has its code and message and comes before any device use."""
import ctypes as C
import struct

import numpy as np
import pytest

import neon_cuda as N

INVALID, UNSUPPORTED = -1, -2
P = 4096  # a pointer that is never followed


def err():
    return N.load().neon_cuda_last_error().decode()


def rope_call(spec=None, type=0, pos=P, n=4, dim=64, targets=None, nt=None, **kw):
    s = N.Rope(64, **kw)._c if spec is None else spec
    t = [(P, 1 << 30, 256, 256, 4)] if targets is None else targets
    arr = struct.pack("%dQ" % (5 * len(t)), *[x or 0 for v in t for x in v])
    return N.load().neon_cuda_rope(C.byref(s), type, pos, n, dim, arr, len(t) if nt is None else nt, 0, None)


@pytest.mark.parametrize("kw,word", [
    (dict(base=0.0), "base"), (dict(base=-1.0), "base"), (dict(base=float("inf")), "base"), (dict(scale=0.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(magnitude=float("inf")), "magnitude"), (dict(yarn=1.5, orig_ctx=8), "yarn"),
    (dict(yarn=float("nan"), orig_ctx=8), "yarn"), (dict(yarn=1.0), "orig_ctx"),
    (dict(yarn=1.0, orig_ctx=8, beta_fast=1.0, beta_slow=2.0), "beta"), (dict(yarn=1.0, orig_ctx=8, base=1.0), "base"),
    (dict(factors=np.zeros(32, np.float32)), "factors")])
def test_rope_spec(kw, word):
    assert rope_call(**kw) == INVALID and word in err()


@pytest.mark.parametrize("n_dims", [0, 1, 63, 66, 258])
def test_rope_dims(n_dims):
    s = N.Rope(64)._c
    s.n_dims = n_dims
    assert rope_call(spec=s) == INVALID and "n_dims" in err()


@pytest.mark.parametrize("kw,code,word", [
    (dict(type=2), UNSUPPORTED, "type"), (dict(pos=None), INVALID, "positions"), (dict(nt=0), INVALID, "targets"),
    (dict(nt=5, targets=[(P, 1 << 30, 256, 256, 4)] * 5), INVALID, "targets"),
    (dict(dim=65), INVALID, "head_dim"), (dict(dim=2048), INVALID, "head_dim"),
    (dict(targets=[(None, P, 256, 256, 4)]), INVALID, "null"), (dict(targets=[(P, P, 256, 256, 0)]), INVALID, "heads"),
    (dict(targets=[(P, 1 << 30, 255, 256, 4)]), INVALID, "stride"), (dict(targets=[(P, 1 << 30, 256, 255, 4)]), INVALID, "stride"),
    (dict(targets=[(P + 2, 1 << 30, 256, 256, 4)]), INVALID, "aligned"),
    (dict(targets=[(P, P, 256, 512, 4)]), INVALID, "strides"),
    (dict(targets=[(P, P + 64, 256, 256, 4)]), INVALID, "overlap"),
    (dict(targets=[(P, P + 4 * 200, 512, 512, 4)]), INVALID, "overlap"),
    (dict(targets=[(P, P + 4 * 256, 512, 600, 4)]), INVALID, "overlap")])
def test_rope_arguments(kw, code, word):
    assert rope_call(**kw) == code and word in err()


@pytest.mark.parametrize("second", [
    (P, P, 256, 256, 4),                    # the same rows twice, in place
    (P * 9, P, 256, 256, 4),                # one output of both
    (P, P * 9, 256, 256, 2),                # reads what the first writes
    (P + 4 * 1000, P * 9, 256, 256, 4),     # its last rows
    (P + 4 * 200, P + 4 * 200, 256, 256, 1),
    (P - 4 * 64, P - 4 * 64, 256, 256, 2),  # from before the first
    (P + 4 * 256, P + 4 * 256, 300, 300, 4)])
def test_rope_targets_are_apart(second):
    assert rope_call(targets=[(P, P, 256, 256, 4), second]) == INVALID and "another target" in err()
    assert rope_call(targets=[second, (P * 40, P, 256, 256, 4)]) == INVALID and "another target" in err()


@pytest.mark.parametrize("first,second", [
    ((P, P, 512, 512, 4), (P + 4 * 256, P + 4 * 256, 512, 512, 4)),     # side by side in one buffer
    ((P + 4 * 448, P + 4 * 448, 512, 512, 1), (P, P, 512, 512, 7)),
    ((P, P * 9, 256, 256, 4), (P, P * 20, 256, 256, 4)),                # one input read twice
    ((P, P, 256, 256, 4), (P + 4 * 1024, P + 4 * 1024, 256, 256, 4))])  # one behind the other
def test_rope_targets_side_by_side(first, second):
    """Not refused for their places: the call after them is (n_heads 0)."""
    assert rope_call(targets=[first, second, (P * 50, P * 50, 64, 64, 0)]) == INVALID and "1 to 65535 heads" in err()


def test_rope_of_nothing():
    assert rope_call(n=0, pos=None) == 0


def cache(**kw):
    c = dict(n_kv_head=2, head_dim=64, capacity=96, k=P, v=P * 2, k_scale=P * 3, v_scale=P * 4, tail=P * 5, tail_block=P * 6,
             past=P * 7)
    c.update(kw)
    return N._Kv8(*[c[f] for f, _ in N._Kv8._fields_])


BAD = [(dict(n_kv_head=0), INVALID), (dict(n_kv_head=20000), INVALID), (dict(head_dim=0), UNSUPPORTED),
       (dict(head_dim=24), UNSUPPORTED), (dict(head_dim=272), UNSUPPORTED), (dict(capacity=0), INVALID),
       (dict(capacity=100), INVALID), (dict(capacity=0x80000000), INVALID)] + [
    (dict([(f, None)]), INVALID) for f in ("k", "v", "k_scale", "v_scale", "tail", "tail_block", "past")] + [
    (dict(k=P + 8), INVALID), (dict(v=P + 1), INVALID), (dict(tail=P + 4), INVALID), (dict(k_scale=P + 2), INVALID),
    (dict(past=P + 1), INVALID)]


@pytest.mark.parametrize("bad,code", BAD)
def test_cache_is_checked_everywhere(bad, code):
    L, c = N.load(), C.byref(cache(**bad))
    good = C.byref(cache(k=P * 8, v=P * 9, k_scale=P * 10, v_scale=P * 11, tail_block=P * 13, past=P * 12))
    assert L.neon_cuda_kv8_append(c, P, 128, P, 128, 1, 0, None) == code
    assert L.neon_cuda_kv8_read(c, 0, 1, P, P, None) == code
    assert L.neon_cuda_kv8_attention(c, P, 128, P, 128, 1, 2, 0.0, 0, None, P, 1 << 20, None) == code
    assert L.neon_cuda_kv8_evict(c, P, good, P * 20, 4, 0, 0, None, P, None) == code
    assert L.neon_cuda_kv8_evict(good, P, c, P * 20, 4, 0, 0, None, P, None) == code


def test_append_arguments():
    L, c = N.load(), C.byref(cache())
    f = L.neon_cuda_kv8_append
    assert f(c, P, 128, P, 128, 1, 8, None) == UNSUPPORTED and "type" in err()
    assert f(c, None, 128, P, 128, 1, 0, None) == INVALID and f(c, P, 128, None, 128, 1, 0, None) == INVALID
    assert f(c, P, 127, P, 128, 2, 0, None) == INVALID and "stride" in err()
    assert f(c, P, 128, P, 128, 97, 0, None) == INVALID and "capacity" in err()
    assert f(c, P + 2, 128, P, 128, 1, 0, None) == INVALID and "aligned" in err()
    assert f(c, None, 0, None, 0, 0, 0, None) == 0


def test_read_arguments():
    L, c = N.load(), C.byref(cache())
    assert L.neon_cuda_kv8_read(c, 90, 7, P, P, None) == INVALID and "range" in err()
    assert L.neon_cuda_kv8_read(c, 97, 0, P, P, None) == INVALID
    assert L.neon_cuda_kv8_read(c, 0, 1, P + 2, P, None) == INVALID
    assert L.neon_cuda_kv8_read(c, 0, 0, P, P, None) == 0 and L.neon_cuda_kv8_read(c, 0, 9, None, None, None) == 0


def test_attention_arguments():
    L, c = N.load(), C.byref(cache())
    f = L.neon_cuda_kv8_attention
    b = C.c_size_t()
    assert L.neon_cuda_kv8_attention_workspace(c, 4, 6, C.byref(b)) == 0 and b.value > 0
    assert L.neon_cuda_kv8_attention_workspace(c, 4, 6, None) == INVALID
    assert f(c, P, 384, P * 2, 384, 4, 6, 0.0, 0, None, P, b.value - 1, None) == INVALID and "workspace" in err()
    assert f(c, P, 384, P * 2, 384, 4, 6, 0.0, 0, None, P + 8, b.value, None) == INVALID and "16 bytes" in err()
    assert f(c, P, 384, P * 2, 384, 4, 6, 0.0, 0, None, None, b.value, None) == INVALID
    assert f(c, P, 384, P, 384, 4, 6, 0.0, 0, None, P, b.value, None) == INVALID and "same buffer" in err()
    assert f(c, P, 383, P * 2, 384, 4, 6, 0.0, 0, None, P, b.value, None) == INVALID and "stride" in err()
    for qs, o, os in ((384, 64, 384), (384, 4 * 384 - 1, 384), (384, -4 * 384 + 1, 384), (800, 384, 700), (800, 383, 800),
                      (800, 417, 800), (800, -1, 800)):  # o: values from Q's first
        assert f(c, P * 4, qs, P * 4 + 4 * o, os, 4, 6, 0.0, 0, None, P, b.value, None) == INVALID and "not overlap" in err()
    assert f(c, P, 384, P * 2, 383, 4, 6, 0.0, 0, None, P, b.value, None) == INVALID and "stride" in err()
    assert f(c, P, 384, P * 2, 384, 4, 5, 0.0, 0, None, P, b.value, None) == INVALID and "n_kv_head" in err()
    assert f(c, P, 384, P * 2, 384, 4, 0, 0.0, 0, None, P, b.value, None) == INVALID
    assert f(c, P, 384, P * 2, 384, 4, 260, 0.0, 0, None, P, b.value, None) == UNSUPPORTED
    assert f(c, P, 384, P * 2, 384, 97, 6, 0.0, 0, None, P, 1 << 40, None) == INVALID and "capacity" in err()
    assert f(c, P, 384, P * 2, 384, 4, 6, float("nan"), 0, None, P, b.value, None) == INVALID and "scale" in err()
    assert f(c, P, 384, P * 2, 384, 4, 6, 0.0, 3, None, P, b.value, None) == UNSUPPORTED
    assert f(c, None, 0, None, 0, 0, 6, 0.0, 0, None, None, 0, None) == 0


def test_evict_arguments():
    L = N.load()
    src = cache()
    other = dict(k=P * 8, v=P * 9, k_scale=P * 10, v_scale=P * 11, tail_block=P * 13, past=P * 12)

    def f(dst=None, keep=8, sink=2, recent=2, w=P, wd=P * 20, kept=P, rope=None):
        return L.neon_cuda_kv8_evict(C.byref(src), w, C.byref(cache(**(other if dst is None else dst))), wd, keep, sink,
                                     recent, rope, kept, None)

    assert f(keep=0) == INVALID and f(keep=97) == INVALID and "keep" in err()
    assert f(sink=9) == INVALID and f(sink=7, recent=2) == INVALID and "sink" in err()
    assert f(w=None) == INVALID and f(wd=None) == INVALID and f(kept=None) == INVALID
    assert f(dst=dict(other, head_dim=128)) == INVALID and f(dst=dict(other, n_kv_head=4)) == INVALID
    for same in ("k", "v", "k_scale", "v_scale", "tail_block", "past"):
        assert f(dst=dict(other, **{same: getattr(src, same)})) == INVALID and "separate" in err()
    assert f(wd=P) == INVALID and "separate" in err()
    assert f(rope=C.byref(N.Rope(128)._c)) == INVALID and "n_dims" in err()
