"""Argument checks of the long-context operators that go by ranges, on a host
without a GPU: overlapping buffers of an eviction."""
import ctypes as C

import pytest

import neon_cuda as N

INVALID = -1
P = 1 << 20  # pointers that are never followed, far apart
H, D, CAP = 2, 64, 96
SIZES = dict(k=H * CAP * D, v=H * CAP * D, k_scale=H * CAP // 8, v_scale=H * CAP // 8, tail=4 * H * 32 * D * 4,
             tail_block=H * 16, past=4)


def cache(at, **kw):
    b = {name: at + i * P for i, name in enumerate(SIZES)}
    b.update(kw)
    return N._Kv8(H, D, CAP, *b.values()), b


def evict(src, dst, w=40 * P, wd=41 * P, kept=42 * P, keep=64):
    return N.load().neon_cuda_kv8_evict(C.byref(src), w, C.byref(dst), wd, keep, 2, 2, None, kept, None)


def err():
    return N.load().neon_cuda_last_error().decode()


WRITTEN = ("k", "v", "k_scale", "v_scale", "tail_block", "past")


@pytest.mark.parametrize("name", WRITTEN + ("wd", "kept"))
@pytest.mark.parametrize("other", WRITTEN + ("w",))
def test_an_output_inside_an_input(name, other):
    src, s = cache(P)
    size = dict(SIZES, w=H * CAP * 4)[other]
    mine = dict(SIZES, wd=H * CAP * 4, kept=H * 64 * 4)[name]
    start = dict(s, w=40 * P)[other]
    for at in (start, start + (size - 1) // 16 * 16, start - (mine - 1) // 16 * 16):  # on 16 bytes
        kw = {name: at}
        dst, _ = cache(20 * P, **({name: at} if name in SIZES else {}))
        assert evict(src, dst, **({} if name in SIZES else kw)) == INVALID and "separate" in err()


@pytest.mark.parametrize("a,b", [("k", "v"), ("k", "k_scale"), ("v", "tail_block"), ("k_scale", "v_scale"), ("past", "tail_block")])
def test_outputs_inside_one_another(a, b):
    src, _ = cache(P)
    _, d = cache(20 * P)
    dst, _ = cache(20 * P, **{a: d[b]})
    assert evict(src, dst) == INVALID and "separate" in err()
    assert evict(src, cache(20 * P)[0], wd=d["k"] + 16) == INVALID and "separate" in err()
    assert evict(src, cache(20 * P)[0], kept=d["v"] + 16) == INVALID and "separate" in err()
    assert evict(src, cache(20 * P)[0], wd=41 * P, kept=41 * P + 16) == INVALID and "separate" in err()


@pytest.mark.parametrize("at", [1, 8])
def test_buffers_side_by_side_are_separate(at):
    """Not refused for their places: all buffers of both caches packed into one allocation (the call fails later,
    for want of a device)."""
    b, p = {}, 64 * P * at
    for side in "sd":
        for name, size in SIZES.items():
            b[side + name] = p
            p += (size + 15) // 16 * 16
    src, dst = (N._Kv8(H, D, CAP, *[b[side + n] for n in SIZES]) for side in "sd")
    assert evict(src, dst, w=p, wd=p + H * CAP * 4, kept=p + 2 * H * CAP * 4) != 0 and "separate" not in err()
    one_tail = N._Kv8(H, D, CAP, *[b["s" + n if n == "tail" else "d" + n] for n in SIZES])
    assert evict(src, one_tail, w=p, wd=p + H * CAP * 4, kept=p + 2 * H * CAP * 4) != 0 and "separate" not in err()


@pytest.mark.parametrize("kw", [dict(base=1e-300, scale=1e-300), dict(base=1e-308, scale=1e-10), dict(scale=5e-324),
                                dict(magnitude=1e39)])
def test_rotations_beyond_the_range_of_numbers(kw):
    """Finite arguments whose frequencies, or whose magnitude in fp32, are not: refused, where every value came out as
    not a number."""
    import struct

    t = struct.pack("5Q", P, 2 * P, 256, 256, 4)
    r = N.Rope(64, **kw)
    assert N.load().neon_cuda_rope(r._ref, 0, P, 4, 64, t, 1, 0, None) == INVALID
    assert "rope: a frequency" in err() or "finite in fp32" in err()


@pytest.mark.parametrize("kw", [dict(base=1e300), dict(base=1e-3), dict(scale=1e300), dict(magnitude=3e38)])
def test_rotations_within_it(kw):
    import struct

    t = struct.pack("5Q", P, 2 * P, 256, 256, 4)
    N.load().neon_cuda_rope(N.Rope(64, **kw)._ref, 0, P, 4, 64, t, 1, 0, None)
    assert "rope" not in err()  # (what it says is that there is no device buffer)
