"""Rotary positions (neon_cuda_rope) against the formula in 64 bits: layouts,
partial heads, scaling, far positions, strides, in place, types, the gradient.

Tolerance, per value: the rotation of a pair (p, q) with |p|, |q| <= r in fp32
is off by at most three roundings of size 2^-24 * 2 r (two products, one sum)
plus the error of cos and sin: the angle's fp32 reduction (half a turn holds
2^-25 of a turn: 2 pi 2^-25 r), sincospif (2 ulp: 2^-23 r) and the magnitude's
product (2^-24 r): below 2^-20 r m in all. Rounding to the type adds half a step."""
import math

import numpy as np
import pytest

import neon_cuda as N

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
TYPES = {"f32": (N.GGML_F32, "float32"), "f16": (N.GGML_F16, "float16"), "bf16": (N.GGML_BF16, "bfloat16")}


@pytest.fixture(scope="module", autouse=True)
def device():
    assert torch.cuda.is_available()
    N.init(0)


def frequencies(n_dims, base, scale=1.0, yarn=0.0, orig=0, fast=32.0, slow=1.0, freq_dim=0, factors=None):
    f = []
    for i in range(n_dims // 2):
        v = base ** (-2.0 * i / (freq_dim or n_dims)) / (1.0 if factors is None else float(factors[i]))
        own = 0.0
        if yarn:
            lo = max(0.0, math.floor(n_dims * math.log(orig / (2 * math.pi * fast)) / (2 * math.log(base))))
            hi = min(n_dims - 1.0, math.ceil(n_dims * math.log(orig / (2 * math.pi * slow)) / (2 * math.log(base))))
            own = yarn * (1 - min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001))))
        f.append(v / scale * (1 - own) + v * own)
    return np.array(f)


def rotated(x, pos, freqs, half, mag=1.0, back=False):
    """x [n, heads, dim] in float64."""
    y = x.astype(np.float64).copy()
    r = 2 * len(freqs)
    a = pos.astype(np.float64)[:, None] * freqs
    c, s = mag * np.cos(a)[:, None], mag * np.sin(a)[:, None] * (-1 if back else 1)
    ia, ib = (np.arange(r // 2), np.arange(r // 2) + r // 2) if half else (np.arange(0, r, 2), np.arange(1, r, 2))
    p, q = x[..., ia].astype(np.float64), x[..., ib].astype(np.float64)
    y[..., ia], y[..., ib] = p * c - q * s, p * s + q * c
    return y


def close(got, want, x, mag, kind, turns=0.0):
    """got within the tolerance of want (the module's docstring); ``turns``: the
    largest angle, of which both sides' 64-bit products lose up to 2^-51."""
    dt = getattr(torch, TYPES[kind][1])
    eps = torch.finfo(dt).eps
    r = np.abs(x).max()
    tol = (2.0 ** -20 + 2.0 ** -51 * turns) * r * abs(mag) + (np.abs(want) * (1 + 2.0 ** -10) * eps / 2 + torch.finfo(dt).smallest_normal * eps
                                       if kind != "f32" else 0.0)
    d = np.abs(got.double().cpu().numpy() - want)
    assert (d <= tol).all(), (d - tol).max()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("n,heads,dim,rot", [(1, 1, 2, 2), (1, 3, 64, 64), (5, 4, 128, 96), (33, 2, 80, 22),
                                             (130, 7, 256, 256), (3, 70, 96, 64)])
def test_layouts_and_sizes(kind, half, n, heads, dim, rot):
    typ, dt = TYPES[kind]
    g = torch.Generator().manual_seed(n * 31 + dim + rot)
    q = torch.randn(n, heads, dim, generator=g).to(getattr(torch, dt))
    k = torch.randn(n, 2, dim, generator=g).to(getattr(torch, dt))
    pos = torch.randint(0, 5000, (n,), generator=g, dtype=torch.int32)
    dq, dk, dp = q.cuda(), k.cuda(), pos.cuda()
    oq, ok = torch.full_like(dq, 7), torch.full_like(dk, 7)
    N.rope(N.Rope(rot, half=half, base=1e4), dp, n, dim, [(dq, oq, heads), (dk, ok, 2)], type=typ)
    f = frequencies(rot, 1e4)
    for x, o in ((q, oq), (k, ok)):
        xd = x.double().numpy()
        close(o, rotated(xd, pos.numpy(), f, half), xd, 1.0, kind)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("spec", [dict(scale=8.0), dict(scale=16.0, yarn=1.0, orig=4096), dict(scale=4.0, yarn=0.5, orig=512, fast=16.0),
                                  dict(freq_dim=128), dict(factors=True), dict(scale=0.5)])
def test_scaling_and_far_positions(half, spec):
    n, dim, rot = 9, 96, 64
    spec = dict(spec)
    g = torch.Generator().manual_seed(5)
    x = torch.randn(n, 3, dim, generator=g)
    pos = torch.tensor([0, 1, -1, 4095, 1 << 20, 2 ** 31 - 1, -2 ** 31, 123456789, 77], dtype=torch.int32)
    if spec.get("factors"):
        spec["factors"] = np.linspace(1, 40, rot // 2).astype(np.float32)
    r = N.Rope(rot, half=half, base=5e5, scale=spec.get("scale", 1.0), yarn=spec.get("yarn", 0.0),
               orig_ctx=spec.get("orig", 0), beta_fast=spec.get("fast", 32.0), magnitude=1.25,
               freq_dim=spec.get("freq_dim", 0), factors=spec.get("factors"))
    f = frequencies(rot, 5e5, **spec)
    dx, out = x.cuda(), torch.empty(n, 3, dim, device="cuda")
    N.rope(r, pos.cuda(), n, dim, [(dx, out, 3)])
    close(out, rotated(x.double().numpy(), pos.numpy(), f, half, 1.25), x.numpy(), 1.25, "f32", 2.0 ** 31 * f.max())


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("half", [False, True])
def test_in_place_strided_and_unaligned(kind, half):
    """Queries and keys inside one projection buffer, rotated where they are; the V part and the rest stay."""
    typ, dt = TYPES[kind]
    n, dim, qh, kh = 17, 64, 4, 2
    stride = (qh + 2 * kh) * dim + 3  # rows not on 16 bytes
    g = torch.Generator().manual_seed(6)
    buf = torch.randn(n, stride, generator=g).to(getattr(torch, dt))
    pos = torch.arange(100, 100 + n, dtype=torch.int32)
    d = buf.cuda()
    q, k = d[:, :qh * dim], d[:, qh * dim:(qh + kh) * dim]
    N.rope(N.Rope(dim, half=half), pos.cuda(), n, dim,
           [(q, q, qh, stride, stride), (k, k, kh, stride, stride)], type=typ)
    f = frequencies(dim, 1e4)
    x = buf[:, :(qh + kh) * dim].reshape(n, qh + kh, dim).double().numpy()
    close(d[:, :(qh + kh) * dim].reshape(n, qh + kh, dim), rotated(x, pos.numpy(), f, half), x, 1.0, kind)
    assert torch.equal(d[:, (qh + kh) * dim:].cpu(), buf[:, (qh + kh) * dim:])


@pytest.mark.parametrize("half", [False, True])
def test_backward_is_the_gradient(half):
    """The transposed rotation: equal to the formula's, and <R x, y> = <x, R^T y> by differences."""
    n, dim, rot = 6, 64, 48
    g = torch.Generator().manual_seed(7)
    x, gy = torch.randn(n, 2, dim, generator=g), torch.randn(n, 2, dim, generator=g)
    pos = torch.randint(0, 1000, (n,), generator=g, dtype=torch.int32)
    r = N.Rope(rot, half=half, magnitude=0.75)
    gx = torch.empty(n, 2, dim, device="cuda")
    N.rope(r, pos.cuda(), n, dim, [(gy.cuda(), gx, 2)], backward=True)
    f = frequencies(rot, 1e4)
    close(gx, rotated(gy.double().numpy(), pos.numpy(), f, half, 0.75, back=True) , gy.numpy(), 0.75, "f32")
    # the loss sum(gy * R x) is linear in x: its difference along any step is gx's product with the step
    step = torch.randn(n, 2, dim, generator=g)
    y0, y1 = torch.empty_like(gx), torch.empty_like(gx)
    N.rope(r, pos.cuda(), n, dim, [(x.cuda(), y0, 2)])
    N.rope(r, pos.cuda(), n, dim, [((x + step).cuda(), y1, 2)])
    got = ((y1 - y0).double().cpu() * gy.double()).sum().item()
    want = (gx.double().cpu() * ((x + step).double() - x.double())).sum().item()
    size = (gy.double().abs() * (x.abs() + step.abs()).double()).sum().item()
    assert abs(got - want) <= 2 * 2.0 ** -19 * size


def test_graph_reads_positions_at_replay():
    n, dim = 3, 128
    x = torch.randn(n, 2, dim, generator=torch.Generator().manual_seed(8))
    d, out, pos = x.cuda(), torch.empty(n, 2, dim, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda")
    r = N.Rope(dim)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        N.rope(r, pos, n, dim, [(d, out, 2)], stream=torch.cuda.current_stream())
    for p in (4, 90000):
        pos.fill_(p)
        g.replay()
        close(out, rotated(x.double().numpy(), np.full(n, p), frequencies(dim, 1e4), False), x.numpy(), 1.0, "f32")
