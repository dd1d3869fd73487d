"""The 8-bit KV cache next to the library's other calls, and what its append
leaves alone: rows beyond the capacity."""
import numpy as np
import pytest

import kv8_oracle as O
import neon_cuda as N
import synth as S
from test_kv8_gpu import cpu, device, no_device_errors, rows  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def test_dropped_rows_are_no_other_calls_error():
    """neon_cuda_sync reports them, and nothing else does: not a matvec over host buffers, not a model's step."""
    tiny = S.ModelConfig(300, 128, 1, 2, 1, 64, 128, ctx_len=64, rope_base=1e4)
    m = N.Model(tiny, list(S.model_tensors(tiny, seed=3)), kv8=True)
    w = N.TensorInfo("w", (64, 32), N.GGML_Q4_0, S.q4_0_weights(32, 64, 1))
    x, y = np.ones(64, np.float32), np.zeros(32, np.float32)
    N.proj_all_positions(w, x, 64, y, 32, 1)
    first = m.forward([1, 2])
    m.set_length(0)
    c = N.Kv8Cache.empty(1, 64, 32)
    k = rows(40, 1, 64, 1).cuda()
    c.past.fill_(20)
    N.sync()
    c.append(k, k, 30)
    torch.cuda.synchronize()
    again = np.zeros(32, np.float32)
    N.proj_all_positions(w, x, 64, again, 32, 1)
    assert np.array_equal(again, y)
    assert np.array_equal(m.forward([1, 2]), first) and m.length == 2
    with pytest.raises(RuntimeError, match="capacity"):
        N.sync()
    N.sync()


def test_rows_beyond_capacity_touch_nothing():
    """Buffers inside larger ones: the rows before, the other heads' and everything around keep their bytes."""
    H, D, cap, pad = 2, 64, 64, 4096
    g = torch.Generator().manual_seed(3)

    def inside(numel, dtype):
        whole = torch.randint(1, 100, (pad + numel + pad,), generator=g).to(dtype).cuda()
        return whole, whole[pad:pad + numel]

    sizes = dict(k=(H * cap * D, torch.int8), v=(H * cap * D, torch.int8), k_scale=(H * cap // 32, torch.float32),
                 v_scale=(H * cap // 32, torch.float32), tail=(4 * H * 32 * D, torch.float32),
                 tail_block=(4 * H, torch.int32), past=(1, torch.int32))
    whole, part = zip(*[inside(*s) for s in sizes.values()])
    b = dict(zip(sizes, part))
    b["tail_block"].fill_(-1)
    before = [w.clone() for w in whole]
    c = N.Kv8Cache(H, D, cap, *b.values())
    x = rows(80, H, D, 10)
    b["past"].fill_(40)
    c.append(x.cuda(), (-x).cuda(), 64)  # rows 40 .. 103 of 64
    with pytest.raises(RuntimeError, match="capacity"):
        N.sync()
    for name, w, was in zip(sizes, whole, before):
        assert torch.equal(w[:pad], was[:pad]) and torch.equal(w[-pad:], was[-pad:]), name
    for name, sign in (("k", 1), ("v", -1)):
        was = dict(zip(sizes, before))[name][pad:-pad].view(H, cap, D)
        scale = dict(zip(sizes, before))[name + "_scale"][pad:-pad].view(H, 2)
        now, now_scale = b[name].view(H, cap, D), b[name + "_scale"].view(H, 2)
        assert torch.equal(now[:, :32], was[:, :32]) and torch.equal(now_scale[:, 0], scale[:, 0])
        for h in range(H):  # block 1: its earlier rows as their codes say, then the new ones
            held = was[h, 32:40].float().cpu().numpy() * scale[h, 1].item()
            cc, ss = O.quantise(np.concatenate([held, sign * x[:24, h].numpy()]))
            assert np.array_equal(cpu(now[h, 32:]), cc) and now_scale[h, 1].item() == ss[0]


@pytest.mark.parametrize("n,heads", [(200, 4), (1, 4)])
def test_attention_right_behind_its_append(n, heads):
    """An attention launched while the append before it still runs reads that append's scales: each step's block
    scales are others, and the results are those of steps that wait."""
    H, D, steps = 2, 64, 40
    k = [(rows(n, H, D, s) * 2.0 ** (s % 9 - 4)).cuda() for s in range(steps)]
    q = torch.randn(n, heads, D, generator=torch.Generator().manual_seed(1)).cuda()
    runs = []
    for wait in (False, True):
        c = N.Kv8Cache.empty(H, D, 256)
        ws = torch.empty(c.attention_workspace(heads, n), dtype=torch.uint8, device="cuda")
        out = torch.empty(steps, n, heads, D, device="cuda")
        torch.cuda.synchronize()
        for s in range(steps):
            c.append(k[s], k[s], n)
            if wait:
                torch.cuda.synchronize()
            c.attention(q, out[s], n, heads, ws)
            if wait:
                torch.cuda.synchronize()
        runs.append(out)
    assert torch.equal(*runs)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("H,D,heads,cap,n", [(1, 64, 1, 32, 1), (8, 128, 64, 4096, 1), (8, 128, 64, 40000, 4), (1, 256, 9, 70016, 3),
                                             (160, 16, 160, 20000, 1), (1, 64, 1, 1024, 33), (1, 64, 64, 8192, 300),
                                             (8, 128, 64, 8192, 40), (2, 192, 4, 9984, 700), (80, 16, 160, 1056, 17),
                                             (1, 256, 33, 2080, 1)])
def test_workspace_is_enough(kind, H, D, heads, cap, n):
    """A workspace of the size that is asked for, anywhere in a larger buffer: nothing before or behind it is touched,
    and calls of fewer tokens run in it too."""
    typ, dt = {"f32": (N.GGML_F32, torch.float32), "bf16": (N.GGML_BF16, torch.bfloat16)}[kind]
    c = N.Kv8Cache.empty(H, D, cap)
    g = torch.Generator(device="cuda").manual_seed(2)
    for codes, scale in ((c.k, c.k_scale), (c.v, c.v_scale)):
        codes.copy_(torch.randint(-127, 128, codes.shape, generator=g, device="cuda", dtype=torch.int8))
        scale.fill_(0.01)
    size = c.attention_workspace(heads, n)
    whole = torch.empty(size + 8192, dtype=torch.uint8, device="cuda")
    q = torch.randn(n, heads, D, generator=g, device="cuda").to(dt)
    w = torch.zeros(H, cap, device="cuda")
    for m in {n, max(1, n // 2), min(n, 7), 1}:
        assert c.attention_workspace(heads, m) <= size
        for at in (4096, 4096 + 16, 4096 + 1008):
            whole.fill_(0xA5)
            o = torch.empty(m, heads, D, dtype=dt, device="cuda")
            c.past.fill_(cap - m)
            c.attention(q, o, m, heads, whole[at:], type=typ, weight=w, workspace_bytes=size)
            assert torch.isfinite(o).all()
            assert (whole[:at] == 0xA5).all() and (whole[at + size:] == 0xA5).all()
