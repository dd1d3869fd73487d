"""The 8-bit KV cache's attention keeps fp32's bits in every type and at every
length (neon_cuda.h: computed in fp32, rounded once at the end), against
float64 over the same codes.

Tolerance, of an output: fp32 outputs as in test_kv8_gpu.py; those of 16 bits
the same before their rounding, and half a step of their type for it. p is
held in two fp16 terms (2^-22 of itself) in every type, so nothing else is
added for the types of 16 bits."""
import numpy as np
import pytest

import kv8_oracle as O
import neon_cuda as N
from test_kv8_gpu import TYPES, attend, cpu, device, no_device_errors, rows, tolerances  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def once_rounded(kind, want, big, v):
    to, _ = tolerances("f32", want, big, v, np.zeros(1))
    return to + (torch.finfo(getattr(torch, TYPES[kind][1])).eps / 2 * (np.abs(want) + to) if kind != "f32" else 0.0)


def values(c, n, H, D):
    k, v = torch.empty(n, H, D, device="cuda"), torch.empty(n, H, D, device="cuda")
    c.read(0, n, k, v)
    return cpu(k).transpose(1, 0, 2), cpu(v).transpose(1, 0, 2)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("H,D,heads,past,n", [(2, 64, 8, 60, 1), (2, 64, 24, 60, 1), (1, 128, 16, 90, 2),
                                              (1, 48, 10, 60, 2), (1, 256, 12, 60, 1), (2, 64, 8, 60, 30),
                                              (1, 128, 8, 90, 40), (1, 80, 4, 60, 40), (1, 192, 4, 60, 40),
                                              (1, 256, 4, 60, 40)])
def test_probabilities_keep_their_bits(kind, H, D, heads, past, n):
    """Values of one size and either sign: an output far below the values shows how p was rounded, in calls of up
    to 8 rows, of 9 to 32 and of more."""
    g = torch.Generator().manual_seed(D + n)
    k = rows(past + n, H, D, 3)
    v = torch.where(torch.rand(past + n, H, D, generator=g) < 0.5, 1.0, -1.0)
    c = N.Kv8Cache.empty(H, D, 192)
    c.append(k.cuda(), v.cuda(), past + n)
    c.past.fill_(past)
    kn, vn = values(c, past + n, H, D)
    q = (torch.randn(n, heads, D, generator=g) * 0.3).to(getattr(torch, TYPES[kind][1])).cuda()
    want, _, big = O.attention(cpu(q), kn, vn, past, D ** -0.5)
    off = np.abs(cpu(attend(c, q, kind)) - want)
    assert (off <= once_rounded(kind, want, big, vn)).all(), (off / once_rounded(kind, want, big, vn)).max()


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("D", [64, 144])
def test_prompt_sums_do_not_fade(kind, D):
    """A long share of keys per CTA whose first half has values of 1 and whose second half has -1, each of nearly
    the same weight: a sum in which the early ones have faded is not near zero."""
    H, heads, n, past = 1, 64, 300 if D == 64 else 150, 40000
    g = torch.Generator().manual_seed(D)
    k = rows(past + n, H, D, 5)
    v = torch.ones(past + n, H, D)
    v[(past + n) // 2:] = -1.0
    c = N.Kv8Cache.empty(H, D, (past + n + 31) // 32 * 32)
    c.append(k.cuda(), v.cuda(), past + n)
    c.past.fill_(past)
    q = (torch.randn(n, heads, D, generator=g) * 0.05).to(getattr(torch, TYPES[kind][1])).cuda()
    out = attend(c, q, kind).double()
    kk, vv = torch.empty(past + n, H, D, device="cuda"), torch.empty(past + n, H, D, device="cuda")
    c.read(0, past + n, kk, vv)
    kk, vv = kk[:, 0].double(), vv[:, 0].double()
    hidden = torch.ones(n, past + n, dtype=torch.bool, device="cuda").triu(past + 1)
    for j in range(0, heads, 7):
        s = (q[:, j].double() @ kk.T) * D ** -0.5
        want = torch.softmax(s.masked_fill_(hidden, -torch.inf), 1) @ vv
        big = (q[:, j].double().abs() @ kk.abs().T).amax(1) * D ** -0.5
        to = once_rounded(kind, want.cpu().numpy(), big.cpu().numpy(), vv.cpu().numpy())
        assert (np.abs(cpu(out[:, j] - want)) <= to).all(), (np.abs(cpu(out[:, j] - want)) / to).max()


@pytest.mark.parametrize("kind,heads", [("f32", 80), ("f16", 800)])
@pytest.mark.parametrize("D", [16, 144])
def test_token_sums_do_not_fade(kind, heads, D):
    """One token of many KV heads over a long cache: so few shares that a warp would sum 16000 keys in one go. All
    values are alike, and the output is that value."""
    H, cap = 80, (1 << 18) if D == 16 else 1 << 17
    past = cap - 100
    g = torch.Generator(device="cuda").manual_seed(1)
    c = N.Kv8Cache.empty(H, D, cap)
    c.k.copy_(torch.randint(-127, 128, (H, cap, D), generator=g, device="cuda", dtype=torch.int8))
    c.k_scale.fill_(0.01)
    c.v.fill_(127)
    c.v_scale.fill_(1 / 127)
    c.past.fill_(past)
    q = (torch.randn(1, heads, D, generator=g, device="cuda") * 0.2).to(getattr(torch, TYPES[kind][1]))
    out = cpu(attend(c, q, kind))
    value = np.full(out.shape, np.float64(np.float32(127) * np.float32(1 / 127)))
    big = cpu(q.double().abs().sum(-1)) * 1.27 * D ** -0.5
    assert (np.abs(out - value) <= once_rounded(kind, value, big, np.ones(1))).all(), np.abs(out - value).max()


@pytest.mark.parametrize("D", [64, 128, 256])
def test_prompt_sums_are_not_short(D):
    """fp32 prompts over values that are all alike: the mean of the outputs is the value. The products sum the two terms
    of 16 keys at a time, and may cut up to an ulp off of the sum so far, which is 0.72 * 2^-23 of it in the mean: of a
    sum that grows evenly over the 992 keys' 124 steps half as much as 124 such cuts of the whole. 0.4 of that is
    added back, so that at most 0.6 of it stays, and what is rounded to nearest, 16 tiles' sums at most 2^-24 each."""
    H, heads, past, n, cap = 2, 8, 892, 100, 992
    g = torch.Generator().manual_seed(D)
    k, v = rows(past + n, H, D, 7), torch.ones(past + n, H, D)
    c = N.Kv8Cache.empty(H, D, cap)
    c.append(k.cuda(), v.cuda(), past + n)
    c.past.fill_(past)
    q = (torch.randn(n, heads, D, generator=g) * 0.2).cuda()
    out = cpu(attend(c, q, "f32"))
    value = np.float64(np.float32(127) * np.float32(1 / 127))
    most = 124 / 2 * 0.72 * 2.0 ** -23
    assert abs(out.mean() / value - 1) <= 0.6 * most + 2.0 ** -20
