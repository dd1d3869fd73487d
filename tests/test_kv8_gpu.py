"""The KV cache in 8 bits (neon_cuda_kv8_*) against its definition in float64
(kv8_oracle.py): codes and scales bit for bit; attention and weights within a
derived tolerance; eviction's rows and codes bit for bit.

Attention's tolerance. A score is a sum of exact products (fp16 terms of q
times integer codes) in fp32: with q's split to 2^-22 of the row's largest and
at most 32 accumulations that each lose 2^-23 of the sum of magnitudes, it is
off by E = 2^-18 * max_j sum |scale q k|, and with exp2's error each p by E +
2^-20 of itself (types of 16 bits may round p to 2^-11). An output is a
weighted mean of v: off by at most twice that times the largest |v|, and by
its own sum's roundings (chains of at most 64 accumulations: 2^-17); the
output's type adds half a step. A weight is a sum of p: off by twice the
relative error of p, and 2^-20 for its sum."""
import numpy as np
import pytest

import kv8_oracle as O
import neon_cuda as N

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
TYPES = {"f32": (N.GGML_F32, "float32"), "f16": (N.GGML_F16, "float16"), "bf16": (N.GGML_BF16, "bfloat16")}


@pytest.fixture(scope="module", autouse=True)
def device():
    assert torch.cuda.is_available()
    N.init(0)


@pytest.fixture(autouse=True)
def no_device_errors():
    """Every test leaves the device's error word clear: no wait ran out."""
    yield
    N.sync()


def cpu(t):
    return t.double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def rows(n, H, D, seed, kind="f32"):
    g = torch.Generator().manual_seed(seed)
    size = 0.5 + 2 * torch.rand(H, D, generator=g)
    return (torch.randn(n, H, D, generator=g) * size).to(getattr(torch, TYPES[kind][1]))


def junk(c):
    """Every row that was not written is garbage, and every scale NaN."""
    c.k.fill_(127)
    c.v.fill_(-127)
    c.k_scale.fill_(float("nan"))
    c.v_scale.fill_(float("nan"))
    c.tail.fill_(float("nan"))
    return c


def check_codes(c, k, v, n):
    """The cache holds rows k, v [n, H, D] (float32 numpy), bit for bit."""
    for x, codes, scales in ((k, c.k, c.k_scale), (v, c.v, c.v_scale)):
        for h in range(c.n_kv_head):
            cc, ss = O.quantise(x[:n, h])
            assert np.array_equal(cpu(codes[h, :n]), cc)
            got = scales[h, :len(ss)].cpu().numpy()
            assert np.array_equal(got.view(np.uint32)[~np.isnan(ss)], ss.view(np.uint32)[~np.isnan(ss)])
            assert np.array_equal(np.isnan(got), np.isnan(ss))


# ---------------------------------------------------------------------------
# append and read
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,D", [(1, 16), (3, 64), (2, 80), (2, 128), (1, 240), (2, 256)])
def test_append_in_pieces(kind, H, D):
    """Any way of cutting the rows into appends leaves the codes of the rows."""
    typ, _ = TYPES[kind]
    total, cap = 205, 256
    k, v = rows(total, H, D, D + H, kind), rows(total, H, D, D + H + 1, kind)
    kn, vn = k.float().numpy(), v.float().numpy()
    dk, dv = k.cuda(), v.cuda()
    for cuts in ([205], [1] * 70 + [135], [31, 1, 32, 33, 64, 3, 41], [5, 100, 100]):
        c = junk(N.Kv8Cache.empty(H, D, cap))
        at = 0
        for n in cuts:
            c.append(dk[at:], dv[at:], n, type=typ)
            at += n
            c.past += n
        assert at == total
        check_codes(c, kn, vn, total)
        assert (c.k[:, total:] == 127).all() and (c.v[:, total:] == -127).all()  # rows behind stay as they were
        assert torch.isnan(c.k_scale[:, (total + 31) // 32:]).all()
        ko, vo = torch.empty(total, H, D, device="cuda"), torch.empty(total, H, D, device="cuda")
        c.read(0, total, ko, vo)
        for h in range(H):
            assert np.array_equal(ko[:, h].cpu().numpy(), O.values(*O.quantise(kn[:, h])))
            assert np.array_equal(vo[:, h].cpu().numpy(), O.values(*O.quantise(vn[:, h])))
        part = torch.full((7 * H * D + 1,), 9.0, device="cuda")
        c.read(30, 7, None, part[1:])  # a buffer on 4 bytes, K left out
        assert torch.equal(part[1:].view(7, H, D), vo[30:37]) and part[0] == 9


def test_append_repeated_and_rewound():
    """A repeated call gives the same cache; after a rewind the rows that stay are exact
    where their block is still held as it came."""
    H, D = 2, 64
    k, v = rows(400, H, D, 1), rows(400, H, D, 2)
    dk, dv = k.cuda(), v.cuda()
    c = N.Kv8Cache.empty(H, D, 448)
    c.append(dk, dv, 37)
    c.past.fill_(37)
    for _ in range(3):
        c.append(dk[37:], dv[37:], 300)  # blocks 1 .. 10
    check_codes(c, k.numpy(), v.numpy(), 337)
    c.past.fill_(337)
    c.append(dk[337:], dv[337:], 20)  # block 10 goes on, block 11 begins
    check_codes(c, k.numpy(), v.numpy(), 357)
    c.past.fill_(340)  # into block 10, which is still held
    k2 = k.clone()
    k2[340:] = rows(60, H, D, 3)
    d2 = k2.cuda()
    c.append(d2[340:], dv[340:], 5)
    check_codes(c, k2.numpy(), v.numpy(), 345)
    # far back: rows 96 .. 99 of block 3 are only held as codes now, and are what those stand for
    kk, vv = torch.empty(100, H, D, device="cuda"), torch.empty(100, H, D, device="cuda")
    c.read(0, 100, kk, vv)
    k3, v3 = kk.cpu(), vv.cpu()
    c.past.fill_(100)
    new = rows(6, H, D, 4)
    for _ in range(2):
        c.append(new.cuda(), new.cuda(), 6)
    k3, v3 = torch.cat([k3, new]), torch.cat([v3, new])
    for x, codes, scales in ((k3, c.k, c.k_scale), (v3, c.v, c.v_scale)):
        for h in range(H):
            cc, ss = O.quantise(x[96:, h].numpy())
            assert np.array_equal(cpu(codes[h, 96:106]), cc) and scales[h, 3].item() == ss[0]


def test_a_rewound_timeline_is_not_used():
    """A block that a later append rewrote is not taken from the older tail."""
    H, D = 1, 16
    a, b = rows(200, H, D, 5), rows(200, H, D, 6)
    c = N.Kv8Cache.empty(H, D, 256)
    c.append(a.cuda(), a.cuda(), 70)      # holds block 2 (rows 64 .. 69)
    c.past.fill_(0)
    c.append(b.cuda(), b.cuda(), 130)     # rewrites block 2
    c.past.fill_(80)                      # inside block 2
    kk = torch.empty(80, H, D, device="cuda")
    c.read(0, 80, kk, None)
    c.append(a.cuda(), a.cuda(), 3)
    x = torch.cat([kk.cpu(), a[:3]])
    cc, ss = O.quantise(x[64:, 0].numpy())
    assert np.array_equal(cpu(c.k[0, 64:83]), cc) and c.k_scale[0, 2].item() == ss[0]


def test_append_edge_values():
    """Zeros, tiny and huge values, exact ties, and values that are not finite."""
    H, D = 1, 16
    x = torch.zeros(7 * 32, H, D)
    x[32:64, 0, 3] = 1e-37
    x[64:96] = torch.randn(32, 1, D, generator=torch.Generator().manual_seed(1)) * 1e37
    x[96:128, 0] = (torch.arange(32 * 16).reshape(32, 16) % 255 - 127) * 0.5  # steps of 1/2 (scale 1/2: whole codes)
    x[96, 0, 0] = 63.5
    x[128:160, 0] = (torch.arange(32 * 16).reshape(32, 16) % 254 - 127).float() + 0.5  # ties at scale 1
    x[128, 0, 0] = 127.0
    x[160, 0, 5] = float("inf")
    x[192, 0, 5] = float("nan")
    c = N.Kv8Cache.empty(H, D, 256)
    c.append(x.cuda(), -x.cuda(), len(x))
    check_codes(c, x.numpy(), -x.numpy(), len(x))
    assert c.k_scale[0, 0] == 0 and c.k_scale[0, 4] == 1


def test_append_strided_and_unaligned():
    H, D = 2, 64
    for kind in ("f32", "bf16"):
        typ, dt = TYPES[kind]
        g = torch.Generator().manual_seed(9)
        buf = torch.randn(50, 2 * H * D + 5, generator=g).to(getattr(torch, dt)).cuda()
        k, v = buf[:, 1:], buf[:, 1 + H * D:]
        c = N.Kv8Cache.empty(H, D, 64)
        c.append(k, v, 50, type=typ, k_stride=buf.stride(0), v_stride=buf.stride(0))
        kn = buf[:, 1:1 + H * D].float().cpu().numpy().reshape(50, H, D)
        vn = buf[:, 1 + H * D:1 + 2 * H * D].float().cpu().numpy().reshape(50, H, D)
        check_codes(c, kn, vn, 50)


def test_rows_beyond_capacity_are_dropped_and_reported():
    H, D = 2, 64
    k = rows(80, H, D, 10)
    c = N.Kv8Cache.empty(H, D, 64)
    guard = c.k.clone()
    c.past.fill_(40)
    N.sync()
    c.append(k.cuda(), k.cuda(), 64)  # rows 40 .. 103
    with pytest.raises(RuntimeError, match="capacity"):
        N.sync()
    N.sync()  # reported once
    cc, ss = O.quantise(np.concatenate([np.zeros((8, D), np.float32), k[:24, 1].numpy()]))
    assert np.array_equal(cpu(c.k[1, 32:64]), cc)
    for past in (64, 2 ** 31 - 1, -1, -2 ** 31):
        c.past.fill_(past)
        before = c.k.clone()
        c.append(k.cuda(), k.cuda(), 1)
        with pytest.raises(RuntimeError, match="capacity"):
            N.sync()
        assert torch.equal(before, c.k)
    assert guard.shape == c.k.shape


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

def filled(H, D, n, cap, seed, kind="f32"):
    """A cache with n rows, garbage behind them, and its values [H, n, D]."""
    c = junk(N.Kv8Cache.empty(H, D, cap))
    if n:
        typ, _ = TYPES[kind]
        c.append(rows(n, H, D, seed, kind).cuda(), rows(n, H, D, seed + 1, kind).cuda(), n, type=typ)
    k, v = torch.empty(n, H, D, device="cuda"), torch.empty(n, H, D, device="cuda")
    c.read(0, n, k, v)
    return c, cpu(k).transpose(1, 0, 2), cpu(v).transpose(1, 0, 2)


def tolerances(kind, out, big, v, w):
    eps = torch.finfo(getattr(torch, TYPES[kind][1])).eps
    e = 2.0 ** -18 * big + 2.0 ** -20 + (2.0 ** -11 if kind != "f32" else 0.0)
    to = (2 * e + 2.0 ** -17)[..., None] * np.abs(v).max(initial=0.0)
    to = to + (eps / 2 * (np.abs(out) + to) if kind != "f32" else 0.0)
    return to, (2 * e.max(initial=0.0) + 2.0 ** -20) * w


def attend(c, q, kind, weight=None, scale=0.0, **kw):
    n, heads, D = q.shape
    o = torch.full_like(q, 7)
    ws = torch.full((c.attention_workspace(heads, n),), 255, dtype=torch.uint8, device="cuda")
    c.attention(q, o, n, heads, ws, type=TYPES[kind][0], weight=weight, scale=scale, **kw)
    return o


def check_attention(H, D, heads, past, n, kind, cap=None, scale=0.0, seed=0, q=None):
    cap = cap or (past + n + 31) // 32 * 32 + 64
    c, k, v = filled(H, D, past + n, cap, seed + past, kind)
    c.past.fill_(past)
    if q is None:
        q = (torch.randn(n, heads, D, generator=torch.Generator().manual_seed(seed + 77)) * 0.7)
    q = q.to(getattr(torch, TYPES[kind][1])).cuda()
    w = torch.full((H, cap), 3.0, device="cuda")
    o = attend(c, q, kind, weight=w, scale=scale)
    want, ww, big = O.attention(cpu(q), k, v, past, scale or D ** -0.5)
    to, tw = tolerances(kind, want, big, v, ww)
    assert (np.abs(cpu(o) - want) <= to).all(), (np.abs(cpu(o) - want) / to).max()
    ww[:, :past] += 3.0  # rows of before are added to, new ones written, the others left
    assert (np.abs(cpu(w[:, :past + n]) - ww) <= tw + 2.0 ** -23 * 4).all()
    assert (w[:, past + n:] == 3).all()
    same = torch.equal(o, attend(c, q, kind, scale=scale))
    assert same  # with or without the weights, again and again: the same bits
    return c, q, o


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,D,heads", [(1, 16, 1), (2, 64, 4), (2, 80, 6), (2, 128, 16), (1, 128, 5), (3, 96, 3),
                                       (1, 256, 2), (2, 192, 24)])
@pytest.mark.parametrize("past,n", [(0, 1), (31, 1), (32, 1), (700, 1), (0, 5), (30, 3), (517, 4)])
def test_attention_of_few_tokens(kind, H, D, heads, past, n):
    check_attention(H, D, heads, past, n, kind)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,D,heads,past,n", [(2, 128, 4, 0, 130), (1, 64, 8, 0, 257), (2, 64, 2, 300, 65),
                                              (1, 128, 3, 33, 200), (1, 80, 2, 95, 129), (1, 256, 2, 20, 140),
                                              (1, 128, 1, 1, 300), (2, 112, 10, 64, 64), (1, 16, 2, 40, 70),
                                               (2, 48, 4, 0, 90), (1, 144, 3, 64, 50), (1, 192, 2, 31, 97),
                                               (1, 240, 4, 10, 33), (1, 128, 64, 77, 1), (2, 64, 24, 500, 3)])
def test_attention_of_prompts(kind, H, D, heads, past, n):
    check_attention(H, D, heads, past, n, kind)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("H,D,heads,past,n", [(2, 64, 22, 400, 1), (1, 48, 9, 5000, 1), (1, 128, 32, 3000, 1),
                                              (1, 256, 31, 900, 1), (1, 64, 3, 20, 3), (1, 16, 16, 33, 2),
                                              (3, 112, 51, 31, 1), (1, 64, 1, 0, 17), (150, 16, 1350, 70, 1)])
def test_attention_of_shared_passes(kind, H, D, heads, past, n):
    """9 to 32 rows of a KV head in 16 bits: sixteen share a pass."""
    check_attention(H, D, heads, past, n, kind)


@pytest.mark.parametrize("past,cap", [(5000, 6016), (3, 8192), (8000, 8032)])
def test_attention_long(past, cap):
    check_attention(2, 64, 8, past, 1, "f32", cap=cap)


def test_attention_scales():
    check_attention(1, 64, 2, 100, 2, "f32", scale=-0.3)
    check_attention(1, 64, 2, 100, 2, "f32", scale=40.0)   # nearly one-hot
    check_attention(1, 64, 2, 100, 2, "f32", scale=1e-30)  # the mean
    check_attention(1, 64, 2, 100, 130, "f32", scale=40.0)


@pytest.mark.parametrize("n", [1, 150])
def test_values_of_very_different_sizes(n):
    """Blocks of V whose scales differ by 10^6 both ways: the output keeps its accuracy relative to its largest block."""
    H, D, past = 1, 64, 200
    k, v = rows(past + n, H, D, 20), rows(past + n, H, D, 21)
    v[32:64] *= 1e-6
    v[64:96] *= 1e6
    v[96:128] = 0
    c = N.Kv8Cache.empty(H, D, 384)
    c.append(k.cuda(), v.cuda(), past + n)
    c.past.fill_(past)
    kk, vv = torch.empty(past + n, H, D, device="cuda"), torch.empty(past + n, H, D, device="cuda")
    c.read(0, past + n, kk, vv)
    q = torch.randn(n, 2, D, generator=torch.Generator().manual_seed(3)).cuda()
    o = attend(c, q, "f32")
    kn, vn = cpu(kk).transpose(1, 0, 2), cpu(vv).transpose(1, 0, 2)
    want, _, big = O.attention(cpu(q), kn, vn, past, D ** -0.5)
    to, _ = tolerances("f32", want, big, vn, np.zeros(1))
    assert (np.abs(cpu(o) - want) <= to).all()
    # queries that see only the small block's neighbourhood: past = 40 hides the large blocks
    c.past.fill_(40)
    o = attend(c, q[:1].contiguous(), "f32")
    want, _, big = O.attention(cpu(q[:1]), kn[:, :41], vn[:, :41], 40, D ** -0.5)
    to, _ = tolerances("f32", want, big, vn[:, :41], np.zeros(1))
    assert (np.abs(cpu(o) - want) <= to).all()


@pytest.mark.parametrize("n", [3, 140])
def test_not_finite_stays_in_its_rows(n):
    """A query that is not finite spoils its own row; a cached row that is not finite, those that attend to its block."""
    H, D, past = 2, 64, 32
    k, v = rows(past + n, H, D, 30), rows(past + n, H, D, 31)
    k[past + 2, 1] = float("nan")  # block 1 of KV head 1: seen from token 0 on
    q = torch.randn(n, 4, D, generator=torch.Generator().manual_seed(4))
    q[1, 0, 5] = float("nan")
    q[2, 1, 5] = float("inf")
    clean = torch.nan_to_num(q, nan=1.0, posinf=1.0)
    c, d = N.Kv8Cache.empty(H, D, 224), N.Kv8Cache.empty(H, D, 224)
    c.append(k.cuda(), v.cuda(), past + n)
    d.append(torch.nan_to_num(k, nan=1.0).cuda(), v.cuda(), past + n)
    c.past.fill_(past)
    d.past.fill_(past)
    w = torch.zeros(H, 224, device="cuda")
    o, ref = attend(c, q.cuda(), "f32", weight=w), attend(d, clean.cuda(), "f32")
    # a weight is not a number where such a query sees the row: those of tokens 1 and 2 see up to row past + 2
    assert torch.isnan(w[0, :past + 3]).all() and torch.isfinite(w[0, past + 3:]).all() and torch.isnan(w[1, :past + n]).all()
    assert torch.isnan(o[:, 2:]).all()            # KV head 1: every token sees block 1
    assert torch.isnan(o[1, 0]).all() and torch.isnan(o[2, 1]).all()
    fine = torch.ones(n, 2, dtype=torch.bool, device="cuda")
    fine[1, 0] = fine[2, 1] = False
    assert torch.equal(o[:, :2][fine], ref[:, :2][fine])
    # a block that only later tokens see leaves the earlier ones alone
    if n > 40:
        k[past + 2, 1] = 1.0
        k[past + 40, 1] = float("nan")  # block 2: rows 64 .., seen from token 32 on
        c.append(k.cuda()[past:], v.cuda()[past:], n)
        o = attend(c, clean.cuda(), "f32")
        assert torch.isnan(o[32:, 2:]).all() and torch.isfinite(o[:32]).all() and torch.isfinite(o[:, :2]).all()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("scale", [0.0, -0.3, 40.0, 1e-30])
def test_shared_passes_of_odd_values(kind, scale):
    """Sixteen rows a pass: scales of scores, blocks of V of very different sizes and one of zeros, scores that rise
    along the cache, and a query row that is not a number, which spoils itself and what it sees of the weights."""
    H, D, heads, past, n = 2, 64, 10, 500, 3
    k, v = rows(past + n, H, D, 20), rows(past + n, H, D, 21)
    k *= torch.linspace(0.05, 3.0, past + n)[:, None, None]
    v[32:64] *= 1e-6
    v[64:96] *= 1e3
    v[96:128] = 0
    c = junk(N.Kv8Cache.empty(H, D, 640))
    c.append(k.cuda(), v.cuda(), past + n)
    c.past.fill_(past)
    kk, vv = torch.empty(past + n, H, D, device="cuda"), torch.empty(past + n, H, D, device="cuda")
    c.read(0, past + n, kk, vv)
    q = torch.randn(n, heads, D, generator=torch.Generator().manual_seed(3)).to(getattr(torch, TYPES[kind][1])).cuda()
    w = torch.zeros(H, 640, device="cuda")
    o = attend(c, q, kind, weight=w, scale=scale)
    kn, vn = cpu(kk).transpose(1, 0, 2), cpu(vv).transpose(1, 0, 2)
    want, ww, big = O.attention(cpu(q), kn, vn, past, scale or D ** -0.5)
    to, tw = tolerances(kind, want, big, vn, ww)
    assert (np.abs(cpu(o) - want) <= to).all()
    assert (np.abs(cpu(w[:, :past + n]) - ww) <= tw + 2.0 ** -23).all()
    bad = q.clone()
    bad[1, 2, 7] = float("nan")  # token 1, KV head 0
    w.zero_()
    p = attend(c, bad, kind, weight=w, scale=scale)
    assert torch.isnan(p[1, 2]).all()
    fine = torch.ones(n, heads, dtype=torch.bool, device="cuda")
    fine[1, 2] = False
    assert torch.equal(p[fine], o[fine])
    assert torch.isnan(w[0, :past + 2]).all() and torch.isfinite(w[0, past + 2:]).all() and torch.isfinite(w[1]).all()


@pytest.mark.parametrize("D", [64, 128, 256])
def test_prompts_on_two_streams(D):
    """Prompts with weights on two caches at once, short and long ones mixed: each as alone."""
    H, heads = 2, 8
    jobs = []
    for s, (past, n, kind) in enumerate([(500, 300, "f16"), (0, 90, "f32")]):
        c, _, _ = filled(H, D, past + n, 832, 30 + s, kind)
        c.past.fill_(past)
        q = torch.randn(n, heads, D, generator=torch.Generator().manual_seed(s)).to(getattr(torch, TYPES[kind][1])).cuda()
        w = torch.zeros(H, 832, device="cuda")
        alone = attend(c, q, kind, weight=w)
        ws = torch.empty(c.attention_workspace(heads, n), dtype=torch.uint8, device="cuda")
        jobs.append((c, q, n, kind, alone, w, torch.empty_like(q), torch.zeros_like(w), ws, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(10):
        for c, q, n, kind, _, _, o, w, ws, st in jobs:
            with torch.cuda.stream(st):
                w.zero_()
            c.attention(q, o, n, heads, ws, type=TYPES[kind][0], weight=w, stream=st)
    torch.cuda.synchronize()
    for _, _, _, _, alone, w, o, got, _, _ in jobs:
        assert torch.equal(o, alone) and torch.equal(got, w)


def test_prompts_in_graphs_that_share_a_workspace():
    """Two captured prompts with weights, replayed in turn over one workspace, at lengths other than the captured."""
    H, D, heads, n = 2, 64, 4, 70
    c, k, v = filled(H, D, 400, 512, 9, "bf16")
    q = torch.randn(2, n, heads, D, generator=torch.Generator().manual_seed(6)).bfloat16().cuda()
    out, weight = torch.empty_like(q), torch.zeros(2, H, 512, device="cuda")
    ws = torch.empty(c.attention_workspace(heads, n), dtype=torch.uint8, device="cuda")
    graphs = []
    c.past.fill_(5)
    for i in range(2):
        c.attention(q[i], out[i], n, heads, ws, type=N.GGML_BF16, weight=weight[i])
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            c.attention(q[i], out[i], n, heads, ws, type=N.GGML_BF16, weight=weight[i], stream=torch.cuda.current_stream())
        graphs.append(g)
    for past in (330, 0, 129):
        c.past.fill_(past)
        weight.zero_()
        for i in (1, 0):
            graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            w = torch.zeros(H, 512, device="cuda")
            assert torch.equal(out[i], attend(c, q[i].contiguous(), "bf16", weight=w)) and torch.equal(weight[i], w)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_a_long_share_of_keys(kind):
    """Many key tiles per CTA, scores that rise along the cache (m moves again and again) and values that agree."""
    H, D, heads, past, n = 1, 64, 2, 7000, 100
    k, v = rows(past + n, H, D, 60), rows(past + n, H, D, 61) + 3.0
    k *= torch.linspace(0.05, 3.0, past + n)[:, None, None]
    c = junk(N.Kv8Cache.empty(H, D, 7168))
    c.append(k.cuda(), v.cuda(), past + n)
    c.past.fill_(past)
    kk, vv = torch.empty(past + n, H, D, device="cuda"), torch.empty(past + n, H, D, device="cuda")
    c.read(0, past + n, kk, vv)
    q = torch.randn(n, heads, D, generator=torch.Generator().manual_seed(5)).to(getattr(torch, TYPES[kind][1])).cuda()
    w = torch.zeros(H, 7168, device="cuda")
    o = attend(c, q, kind, weight=w)
    kn, vn = cpu(kk).transpose(1, 0, 2), cpu(vv).transpose(1, 0, 2)
    want, ww, big = O.attention(cpu(q), kn, vn, past, D ** -0.5)
    to, tw = tolerances(kind, want, big, vn, ww)
    assert (np.abs(cpu(o) - want) <= to).all()
    assert (np.abs(cpu(w[:, :past + n]) - ww) <= tw + 2.0 ** -23).all()


def test_offsets_beyond_32_bits():
    """The second head of a cache whose codes fill 2^33 bytes, its last rows: the others are zeros, that weigh 1 each."""
    H, D, cap, n = 2, 256, 1 << 24, 3
    c = N.Kv8Cache.empty(H, D, cap)
    past = cap - n
    c.past.fill_(past)
    k, v = rows(n, H, D, 70), rows(n, H, D, 71)
    c.append(k.cuda(), v.cuda(), n)
    kk, vv = torch.empty(n, H, D, device="cuda"), torch.empty(n, H, D, device="cuda")
    c.read(past, n, kk, vv)
    for h in range(H):  # (the block's earlier rows are zeros)
        want = O.quantise(np.concatenate([np.zeros((29, D), np.float32), k[:, h].numpy()]))
        assert np.array_equal(cpu(c.k[h, past:]), want[0][29:])
    q = torch.randn(n, 2, D, generator=torch.Generator().manual_seed(6)).cuda() * 3
    w = torch.zeros(H, cap, device="cuda")
    o = attend(c, q, "f32", weight=w)
    for t in range(n):
        for h in range(H):
            s = (cpu(kk)[:t + 1, h] @ cpu(q)[t, h]) * D ** -0.5
            p = np.exp(s) / (past + np.exp(s).sum())
            want = p @ cpu(vv)[:t + 1, h]
            assert np.abs(cpu(o[t, h]) - want).max() <= 2.0 ** -10 * np.abs(p[:, None] * cpu(vv)[:t + 1, h]).max() * (t + 1)
    total = 1.0 / (past + np.exp((cpu(kk)[:1, 1] @ cpu(q)[0, 1]) * D ** -0.5).sum())
    assert abs(w[1, 12345].item() / (3 * total) - 1) < 1e-2 and w[1, past - 1].item() > 0
    del c, w
    torch.cuda.empty_cache()


def test_a_prompt_of_tokens_without_rows():
    c, k, v = filled(2, 64, 200, 224, 1)
    q = torch.randn(140, 4, 64, generator=torch.Generator().manual_seed(7)).cuda()
    w = torch.full((2, 224), 3.0, device="cuda")
    c.past.fill_(-20)
    o = attend(c, q, "f32", weight=w)
    assert (o[:20] == 0).all()
    want, ww, big = O.attention(cpu(q[20:]), k[:, :120], v[:, :120], 0, 64 ** -0.5)
    to, tw = tolerances("f32", want, big, v, ww)
    assert (np.abs(cpu(o[20:]) - want) <= to).all()
    assert (np.abs(cpu(w[:, :120]) - ww) <= tw + 2.0 ** -23).all() and (w[:, 120:] == 3).all()
    c.past.fill_(-1000)
    assert (attend(c, q, "f32", weight=w) == 0).all()


def test_no_rows_to_attend_to():
    c, _, _ = filled(2, 64, 40, 64, 1)
    q = torch.randn(5, 4, 64, device="cuda")
    w = torch.full((2, 64), 3.0, device="cuda")
    c.past.fill_(-3)
    o = attend(c, q, "f32", weight=w)
    assert (o[:2] == 0).all() and torch.isfinite(o).all() and (o[2:] != 0).any()
    c.past.fill_(-100)
    assert (attend(c, q, "f32", weight=w) == 0).all()
    assert (w[:, 2:] == 3).all()


def test_strided_queries_and_outputs():
    H, D, heads, past, n = 2, 64, 4, 90, 9
    c, q, o = check_attention(H, D, heads, past, n, "f32")
    buf = torch.zeros(n, heads * D + 3, device="cuda")
    buf[:, 1:1 + heads * D] = q.view(n, -1)
    out = torch.full((n, heads * D + 7), 5.0, device="cuda")
    ws = torch.empty(c.attention_workspace(heads, n), dtype=torch.uint8, device="cuda")
    c.attention(buf[:, 1:], out[:, 2:], n, heads, ws, q_stride=buf.stride(0), o_stride=out.stride(0))
    assert torch.equal(out[:, 2:2 + heads * D].reshape(n, heads, D), o)
    assert (out[:, :2] == 5).all() and (out[:, 2 + heads * D:] == 5).all()


def test_two_streams_and_a_graph():
    """Calls on two caches at once, each with its workspace, and a captured decode step that reads past at replay."""
    H, D, heads = 2, 128, 8
    made = [filled(H, D, 900, 1024, s) for s in (1, 2)]
    qs = [torch.randn(1, heads, D, generator=torch.Generator().manual_seed(s)).cuda() for s in (3, 4)]
    alone = []
    for (c, _, _), q in zip(made, qs):
        c.past.fill_(899)
        alone.append(attend(c, q, "f32"))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    ws = [torch.empty(made[0][0].attention_workspace(heads, 1), dtype=torch.uint8, device="cuda") for _ in range(2)]
    outs = [torch.empty_like(q) for q in qs]
    torch.cuda.synchronize()
    for _ in range(20):
        for (c, _, _), q, st, w, o in zip(made, qs, streams, ws, outs):
            c.attention(q, o, 1, heads, w, stream=st)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], alone[0]) and torch.equal(outs[1], alone[1])

    c, k, v = made[0]
    new = rows(4, H, D, 50).cuda()
    step_k, out = torch.empty(1, H, D, device="cuda"), torch.empty(1, heads, D, device="cuda")
    weight = torch.zeros(H, 1024, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        st = torch.cuda.current_stream()
        c.append(step_k, step_k, 1, stream=st)
        c.attention(qs[0], out, 1, heads, ws[0], weight=weight, stream=st)
        c.past += 1
    c.past.fill_(900)
    weight.zero_()
    e, _, _ = filled(H, D, 900, 1024, 1)
    e.past.fill_(900)
    for t in range(4):
        step_k.copy_(new[t:t + 1])
        g.replay()
        e.append(new[t:t + 1], new[t:t + 1], 1)
        assert torch.equal(out, attend(e, qs[0], "f32"))
        e.past += 1
    assert c.past.item() == 904 and torch.equal(c.k[:, :904], e.k[:, :904])
    assert abs(weight.sum().item() - 4 * heads) < 1e-3


# ---------------------------------------------------------------------------
# eviction
# ---------------------------------------------------------------------------

def check_evict(H, D, length, keep, sink, recent, w, cap=None, dcap=None, rope=None):
    cap = cap or (length + 31) // 32 * 32 + 32
    c, k, v = filled(H, D, length, cap, length + D)
    c.past.fill_(length)
    before = c.k.clone(), c.v.clone(), c.k_scale.clone(), c.v_scale.clone()
    W = torch.full((H, cap), 1e9, device="cuda")  # what lies behind the rows does not count
    W[:, :length] = w.cuda()
    d = junk(N.Kv8Cache.empty(H, D, dcap or (keep + 31) // 32 * 32))
    dw = torch.full((H, d.capacity), -1.0, device="cuda")
    kept = torch.full((H, keep), -7, dtype=torch.int32, device="cuda")
    c.evict(d, keep, sink, recent, W, dw, kept, rope=rope)
    m = min(length, keep)
    assert d.past.item() == m and (d.tail_block == -1).all() and c.past.item() == length
    assert torch.equal(c.k, before[0]) and torch.equal(c.v, before[1])
    for h in range(H):
        r = O.evicted(w[h].numpy(), length, keep, sink, recent)
        assert np.array_equal(cpu(kept[h, :m]), r) and (kept[h, m:] == -1).all()
        assert np.array_equal(dw[h, :m].cpu().numpy(), w[h].numpy()[r])
        for name, x in (("k", k), ("v", v)):
            if name == "k" and rope is not None:
                continue
            codes, scales = getattr(c, name)[h, :length].cpu().numpy(), getattr(c, name + "_scale")[h].cpu().numpy()
            cc, ss = O.moved(x[h].astype(np.float32), r, codes, scales)
            assert np.array_equal(cpu(getattr(d, name)[h, :m]), cc)
            assert np.array_equal(getattr(d, name + "_scale")[h, :len(ss)].cpu().numpy(), ss)
    assert (d.v[:, m:] == -127).all() and (dw[:, m:] == -1).all()
    return c, d, k, kept


@pytest.mark.parametrize("H,D", [(1, 16), (2, 64), (3, 80), (2, 128), (1, 256)])
@pytest.mark.parametrize("length,keep,sink,recent", [(100, 50, 4, 10), (100, 99, 0, 0), (33, 32, 32, 0), (33, 32, 0, 32),
                                                     (64, 1, 0, 0), (500, 37, 3, 30), (1000, 513, 4, 64),
                                                     (40, 40, 4, 4), (20, 64, 1, 1), (0, 32, 0, 0)])
def test_evict(H, D, length, keep, sink, recent):
    w = torch.randn(H, length, generator=torch.Generator().manual_seed(length + keep)).exp()
    check_evict(H, D, length, keep, sink, recent, w)


@pytest.mark.parametrize("what", ["equal", "few", "zeros", "specials", "bits"])
def test_evict_ties_and_odd_weights(what):
    H, D, length, keep = 2, 16, 9001, 4000
    g = torch.Generator().manual_seed(3)
    w = {"equal": torch.full((H, length), 0.25), "few": torch.randint(0, 3, (H, length), generator=g).float(),
         "zeros": torch.zeros(H, length), "specials": torch.randn(H, length, generator=g),
         "bits": 1 + torch.randint(0, 300, (H, length), generator=g).float() * 2.0 ** -23}[what]
    if what == "zeros":
        w[:, ::2] = -0.0
    if what == "specials":
        w[:, 5::50] = float("inf")
        w[:, 6::50] = -float("inf")
        w[:, 7::500] = 1e-42
    check_evict(H, D, length, keep, 10, 200, w)


def test_evict_long_and_into_a_larger_cache():
    H, D, length = 1, 64, 70001
    w = torch.randn(H, length, generator=torch.Generator().manual_seed(1)).exp()
    w[:, ::5] = 0.5
    check_evict(H, D, length, 30011, 16, 1000, w, dcap=32000)


def test_evict_keeps_nan_first():
    H, D, length, keep = 1, 16, 200, 40
    w = torch.rand(H, length, generator=torch.Generator().manual_seed(2))
    bad = [50, 90, 91]
    for i, b in enumerate(bad):
        w[0, b] = float("nan") if i != 1 else -float("nan")
    c, k, v = filled(H, D, length, 224, 1)
    c.past.fill_(length)
    d, kept = N.Kv8Cache.empty(H, D, 64), torch.empty(H, keep, dtype=torch.int32, device="cuda")
    W = torch.zeros(H, 224, device="cuda")
    W[:, :length] = w.cuda()
    c.evict(d, keep, 0, 0, W, torch.empty(H, 64, device="cuda"), kept)
    w[0, bad] = 2.0
    assert np.array_equal(cpu(kept[0]), O.evicted(w[0].numpy(), length, keep, 0, 0))


@pytest.mark.parametrize("half", [False, True])
def test_evict_turns_keys(half):
    """With a rotation, K rows move to their new positions: within one code of the formula in 64 bits
    (its rounding may differ where fp32 cos and sin put a value across a tie), relative to the block's scale."""
    H, D, rot, length, keep = 2, 64, 48, 700, 300
    w = torch.randn(H, length, generator=torch.Generator().manual_seed(8)).exp()
    r = N.Rope(rot, half=half, base=5e3, freq_dim=D, magnitude=3.0)  # the magnitude is in the rows already
    c, d, k, kept = check_evict(H, D, length, keep, 4, 100, w, rope=r)
    f = 5e3 ** (-2.0 * np.arange(rot // 2) / D)
    ia, ib = (np.arange(rot // 2), np.arange(rot // 2) + rot // 2) if half else (np.arange(0, rot, 2), np.arange(1, rot, 2))
    for h in range(H):
        kr = cpu(kept[h])
        x = k[h][kr].copy()
        a = (np.arange(keep) - kr)[:, None] * f
        p, q = x[:, ia].copy(), x[:, ib].copy()
        x[:, ia], x[:, ib] = p * np.cos(a) - q * np.sin(a), p * np.sin(a) + q * np.cos(a)
        s = d.k_scale[h].cpu().numpy().astype(np.float64)
        got = cpu(d.k[h, :keep]) * np.repeat(s, 32)[:keep, None]
        top = np.array([np.abs(x[b * 32:(b + 1) * 32]).max() for b in range((keep + 31) // 32)])
        assert np.allclose(s[:len(top)] * 127, top, rtol=2.0 ** -19)
        assert (np.abs(got - x) <= np.repeat(s, 32)[:keep, None] * (0.5 + 2.0 ** -10)).all()


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------

def test_a_conversation():
    """A prompt and decode steps over a cache that is thinned on the way: rotation, append, attention with weights,
    eviction, against the same steps in float64 over the same codes."""
    H, D, heads, cap, keep = 2, 64, 6, 192, 96
    g = torch.Generator().manual_seed(11)
    spec = N.Rope(D, half=True, base=1e4)
    caches = [N.Kv8Cache.empty(H, D, cap), N.Kv8Cache.empty(H, D, cap)]
    weights = [torch.zeros(H, cap, device="cuda"), torch.zeros(H, cap, device="cuda")]
    kept = torch.empty(H, keep, dtype=torch.int32, device="cuda")
    ws = torch.empty(caches[0].attention_workspace(heads, 140), dtype=torch.uint8, device="cuda")
    track = np.zeros((H, 0))  # the weights in float64
    seen = 0
    for n in [140] + [1] * 50 + [3] * 20:
        c, w = caches[0], weights[0]
        if c.past.item() + n > cap:
            c.evict(caches[1], keep, 4, 16, w, weights[1], kept)
            track = np.stack([track[h][cpu(kept[h])] for h in range(H)])
            assert np.array_equal(cpu(kept), np.stack([O.evicted(w[h].cpu().numpy(), cap if n == 1 else c.past.item(), keep, 4, 16)
                                                       for h in range(H)])[:, :keep])
            caches.reverse()
            weights.reverse()
            c, w = caches[0], weights[0]
        past = c.past.item()
        q, k, v = (torch.randn(n, x, D, generator=g).cuda() for x in (heads, H, H))
        pos = torch.arange(seen, seen + n, dtype=torch.int32, device="cuda")
        N.rope(spec, pos, n, D, [(q, q, heads), (k, k, H)])
        c.append(k, v, n)
        o = torch.empty(n, heads, D, device="cuda")
        c.attention(q, o, n, heads, ws, weight=w)
        kk, vv = (torch.empty(past + n, H, D, device="cuda") for _ in range(2))
        c.read(0, past + n, kk, vv)
        kn, vn = cpu(kk).transpose(1, 0, 2), cpu(vv).transpose(1, 0, 2)
        want, ww, big = O.attention(cpu(q), kn, vn, past, D ** -0.5)
        to, _ = tolerances("f32", want, big, vn, ww)
        assert (np.abs(cpu(o) - want) <= to).all()
        track = np.concatenate([track, np.zeros((H, n))], 1) + ww
        assert np.allclose(cpu(w[:, :past + n]), track, rtol=1e-4, atol=1e-5)
        c.past += n
        seen += n
