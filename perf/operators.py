"""The work that the long-context operators are measured on: rotary positions, the KV cache in 8 bits (append and
attention), and eviction from it by accumulated attention weight.

A cache holds, for each KV head, int8 codes [n_kv_head][capacity][head_dim] of K and of V with one fp32 scale for
each block of 32 rows and head: a row's value is the fp32 number code * scale. A block's scale is amax / 127 over the
rows that it holds, its codes are the nearest integers to value / scale (ties to even), and a block without a
value as large as 127 times the smallest normal fp32 number has scale and codes 0. The rows of the block that is being
filled are also held as they came (the tail), so a block's codes depend on its rows and not on how they arrived.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

BLOCK = 32
TINY = 127.0 * float(np.finfo(np.float32).tiny)  # a block below this is held as zeros
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # the query and key heads of one new token, as each decode step rotates them
        {"name": "rope_token", "op": "rope", "n": 1, "heads": 16, "kv_heads": 8, "dim": 128, "rot": 128,
         "half": False, "yarn": False, "scale": 1.0, "base": 1e6, "start": 300, "type": "f32", "back": False},
        # a long prompt's chunk far out in a stretched context: part of each head, halves layout
        {"name": "rope_prompt", "op": "rope", "n": 4099, "heads": 24, "kv_heads": 8, "dim": 128, "rot": 96,
         "half": True, "yarn": True, "scale": 32.0, "base": 1e4, "start": 120000, "type": "bf16", "back": False},
        # one decode step's K and V rows into a block that is partly full
        {"name": "append_token", "op": "append", "n": 1, "past": 1037, "kv_heads": 8, "dim": 128, "type": "f32"},
        # a long prompt's K and V, not starting at a block's edge
        {"name": "append_prompt", "op": "append", "n": 8191, "past": 77, "kv_heads": 8, "dim": 128, "type": "bf16"},
        # a decode step early in a conversation
        {"name": "token", "op": "attend", "n": 1, "past": 511, "heads": 16, "kv_heads": 8, "dim": 128, "type": "f32",
         "weight": False},
        # a decode step with a full long context, the weights of the cached rows accumulated for eviction
        {"name": "token_long", "op": "attend", "n": 1, "past": 131070, "heads": 64, "kv_heads": 8, "dim": 128,
         "type": "f32", "weight": True},
        # a few drafted tokens checked at once
        {"name": "tokens_few", "op": "attend", "n": 3, "past": 20011, "heads": 24, "kv_heads": 8, "dim": 64,
         "type": "bf16", "weight": False},
        # a whole prompt
        {"name": "prompt", "op": "attend", "n": 2048, "past": 0, "heads": 64, "kv_heads": 8, "dim": 128,
         "type": "f32", "weight": False},
        # a longer prompt in 16 bits
        {"name": "prompt_16", "op": "attend", "n": 4096, "past": 0, "heads": 64, "kv_heads": 8, "dim": 128,
         "type": "bf16", "weight": False},
        # one chunk of a document behind a long past, the weights accumulated
        {"name": "chunk", "op": "attend", "n": 501, "past": 30000, "heads": 32, "kv_heads": 4, "dim": 64,
         "type": "f16", "weight": True},
        # making room in a short cache
        {"name": "evict_short", "op": "evict", "past": 1024, "keep": 513, "sink": 4, "recent": 64, "kv_heads": 8,
         "dim": 128},
        # making room in a long one
        {"name": "evict_long", "op": "evict", "past": 131071, "keep": 32768, "sink": 64, "recent": 4096,
         "kv_heads": 8, "dim": 128},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "append", "attend", "attend", "attend", "evict"])
    kv = rng.choice([1, 2, 4, 8])
    dim = rng.choice([64, 64, 128, 128, 128, 80, 96, 256])
    kv = min(kv, 1024 // dim)
    kind = rng.choice(["f32", "f16", "bf16"])
    if op == "rope":
        rot = dim if rng.random() < 0.5 else 2 * rng.randint(8, dim // 2)
        yarn = rng.random() < 0.4
        return {"op": op, "n": _log(rng, 1, 4096), "heads": kv * rng.randint(1, 4), "kv_heads": kv, "dim": dim,
                "rot": rot, "half": rng.random() < 0.5, "yarn": yarn, "scale": rng.choice([1.0, 4.0, 32.0]) if not yarn else 16.0,
                "base": rng.choice([1e4, 5e5, 1e6]), "start": _log(rng, 1, 1000000), "type": kind,
                "back": rng.random() < 0.3}
    if op == "append":
        return {"op": op, "n": _log(rng, 1, 8000), "past": _log(rng, 1, 8000) - 1, "kv_heads": kv, "dim": dim,
                "type": kind}
    if op == "evict":
        past = _log(rng, 64, 100000)
        keep = rng.randint(past // 4, past - 1) if past > 256 else rng.randint(40, past)
        keep = min(keep, 30000)
        sink = rng.randint(0, 16)
        return {"op": op, "past": past, "keep": keep, "sink": sink, "recent": rng.randint(0, min(keep - sink, 512)),
                "kv_heads": kv, "dim": dim}
    n = rng.choice([1, 1, rng.randint(2, 16), _log(rng, 16, 2000)])
    past = _log(rng, 1, 100000 if n <= 16 else 16000) - 1
    heads = kv * rng.choice([1, 2, 3, 4, 5, 8])
    n = max(1, min(n, int(2.5e11 / (4 * dim * heads * (past + n)))))
    return {"op": op, "n": n, "past": past, "heads": heads, "kv_heads": kv, "dim": dim, "type": kind,
            "weight": rng.random() < 0.4}


def _capacity(rows):
    return (rows + BLOCK - 1) // BLOCK * BLOCK + BLOCK


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    H, D = case["kv_heads"], case["dim"]
    s = {"case": case}
    if case["op"] == "rope":
        n, dt = case["n"], DTYPES[case["type"]]
        s["q"] = normal(n, case["heads"], D).to(dt)
        s["k"] = normal(n, H, D).to(dt)
        s["pos"] = torch.arange(case["start"], case["start"] + n, dtype=torch.int32, device="cuda")
        return s
    n = case.get("n", 0)
    rows = case["past"] + n
    C = _capacity(rows)
    # rows as projections give them: normal, each channel of K with its own size
    size = 0.5 + 2 * torch.rand(H, 1, D, generator=g, device="cuda")

    def codes(by):
        c = torch.empty(H, C, D, dtype=torch.int8, device="cuda")
        sc = torch.empty(H, C // BLOCK, device="cuda")
        for h in range(H):
            x = normal(C // BLOCK, BLOCK, D) * (by[h] if by is not None else 1.0)
            a = x.abs().amax(dim=(1, 2))
            sc[h] = a / 127
            c[h] = torch.round(x / sc[h][:, None, None]).clamp_(-127, 127).to(torch.int8).view(C, D)
        return c, sc

    s["k"], s["k_scale"] = codes(size)
    s["v"], s["v_scale"] = codes(None)
    s["past"] = torch.tensor([case["past"]], dtype=torch.int32, device="cuda")
    # the tail: two blocks' rows for K and V; the first slot holds the block that is being filled
    s["tail"] = torch.zeros(2, 2, H, BLOCK, D, device="cuda")
    s["tail_block"] = torch.full((2, H, 2), -1, dtype=torch.int32, device="cuda")
    b0, r0 = divmod(case["past"], BLOCK)
    if r0:
        s["tail_block"][:, :, 0] = b0
        s["tail"][0, 0, :, :r0] = normal(H, r0, D) * size
        s["tail"][1, 0, :, :r0] = normal(H, r0, D)
    if case["op"] == "append":
        dt = DTYPES[case["type"]]
        s["new_k"] = (normal(n, H, D) * size.view(H, D)).to(dt)
        s["new_v"] = normal(n, H, D).to(dt)
    elif case["op"] == "attend":
        # keys are like their queries in part, so that the weights are uneven as a model's are
        s["q"] = (normal(n, case["heads"], D) * 0.7).to(DTYPES[case["type"]])
        if case["weight"]:
            s["weight"] = torch.rand(H, C, generator=g, device="cuda")
    else:
        s["weight"] = (normal(H, C) * 2).exp()
        s["weight"][:, ::7] = 0.125  # many rows of the same weight
        K = _capacity(case["keep"])
        s["dst"] = {"k": torch.zeros(H, K, D, dtype=torch.int8, device="cuda"),
                    "v": torch.zeros(H, K, D, dtype=torch.int8, device="cuda"),
                    "k_scale": torch.zeros(H, K // BLOCK, device="cuda"),
                    "v_scale": torch.zeros(H, K // BLOCK, device="cuda"),
                    "past": torch.zeros(1, dtype=torch.int32, device="cuda"),
                    "tail": torch.zeros(2, 2, H, BLOCK, D, device="cuda"),
                    "tail_block": torch.full((2, H, 2), -1, dtype=torch.int32, device="cuda")}
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------

def _turns(case, device):
    """The rotation of each pair per position, in 64 bits."""
    rot, base, scale = case["rot"], case["base"], case["scale"]
    i = torch.arange(rot // 2, dtype=torch.float64, device=device)
    f = base ** (-2.0 * i / rot)
    if not case["yarn"]:
        return f / scale, 1.0
    at = [rot * math.log(4096 / (b * 2 * math.pi)) / (2 * math.log(base)) for b in (32.0, 1.0)]
    lo, hi = max(0.0, math.floor(at[0])), min(rot - 1.0, math.ceil(at[1]))
    own_part = 1 - ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)  # how far a pair keeps its own frequency
    return f / scale * (1 - own_part) + f * own_part, 0.1 * math.log(scale) + 1.0


def _rope(x, pos, case):
    f, size = _turns(case, x.device)
    a = pos.double()[:, None] * f
    c, s = (size * torch.cos(a)).float()[:, None], (size * torch.sin(a)).float()[:, None]
    if case["back"]:
        s = -s
    r, y = case["rot"], x.float().clone()
    if case["half"]:
        u, v = x[..., :r // 2].float(), x[..., r // 2:r].float()
        y[..., :r // 2], y[..., r // 2:r] = u * c - v * s, u * s + v * c
    else:
        u, v = x[..., 0:r:2].float(), x[..., 1:r:2].float()
        y[..., 0:r:2], y[..., 1:r:2] = u * c - v * s, u * s + v * c
    return y.to(x.dtype)


def _quantised(x):
    """Blocks x[H, b, BLOCK, D] as the values that their 8 bits stand for."""
    a = x.abs().amax(dim=(2, 3), keepdim=True)
    # by a tensor: torch multiplies by a plain number's reciprocal, and a scale is the quotient
    s = torch.where(a >= TINY, a / torch.full_like(a, 127.0), torch.zeros_like(a))
    c = torch.where(s > 0, torch.round(x.double() / torch.where(s > 0, s, torch.ones_like(s)).double()).float(), torch.zeros_like(x))
    return c * s


def _blocks(x):
    H, n, D = x.shape
    b = (n + BLOCK - 1) // BLOCK
    y = torch.zeros(H, b * BLOCK, D, device=x.device)
    y[:, :n] = x
    return y.view(H, b, BLOCK, D)


def _append(s, which, new):
    case = s["case"]
    r0 = case["past"] % BLOCK
    x = torch.cat([s["tail"][which, 0, :, :r0], new.float().transpose(0, 1)], dim=1)
    q = _quantised(_blocks(x))
    return q.reshape(x.shape[0], -1, x.shape[2])[:, :x.shape[1]].transpose(0, 1).contiguous()


def _values(codes, scale, rows):
    return codes[:, :rows].float() * scale.repeat_interleave(BLOCK, dim=1)[:, :rows, None]


def _attend(s):
    case = s["case"]
    n, past, H, D = case["n"], case["past"], case["kv_heads"], case["dim"]
    group, rows = case["heads"] // H, past + n
    k, v = _values(s["k"], s["k_scale"], rows), _values(s["v"], s["v_scale"], rows)
    q = s["q"].float().view(n, H, group, D).permute(1, 0, 2, 3).reshape(H, n * group, D)
    t = torch.matmul(q, k.transpose(1, 2)) * (1 / math.sqrt(D))
    if n > 1:
        later = torch.arange(rows, device=q.device)[None, :] > (past + torch.arange(n, device=q.device))[:, None]
        t.view(H, n, group, rows).masked_fill_(later[None, :, None, :], -math.inf)
    t -= t.amax(dim=2, keepdim=True)
    t.exp_()
    total = t.sum(dim=2, keepdim=True)
    out = torch.matmul(t, v) / total
    out = out.view(H, n, group, D).permute(1, 0, 2, 3).reshape(n, H * group, D).to(s["q"].dtype)
    if not case["weight"]:
        return {"out": out}
    t /= total
    w = s["weight"].clone()
    given = t.sum(dim=1)
    w[:, :past] += given[:, :past]
    w[:, past:rows] = given[:, past:]
    return {"out": out, "weight": w}


def _evict(s):
    case = s["case"]
    L, keep, sink, recent = case["past"], case["keep"], case["sink"], case["recent"]
    H, D = case["kv_heads"], case["dim"]
    w = s["weight"][:, :L]
    m = min(L, keep)
    if L > keep:
        middle = w[:, sink:L - recent]
        # a stable order: the largest weights first, the lowest row first among equals
        order = torch.argsort(middle, dim=1, descending=True, stable=True)[:, :keep - sink - recent] + sink
        ends = torch.cat([torch.arange(sink, device=w.device), torch.arange(L - recent, L, device=w.device)])
        kept = torch.sort(torch.cat([order, ends.expand(H, -1)], dim=1), dim=1).values
    else:
        kept = torch.arange(L, device=w.device).expand(H, -1)
    moved = _blocks((kept != torch.arange(m, device=w.device)).float()[..., None]).sum(dim=(2, 3), keepdim=True) > 0

    def packed(codes, scale):  # a block whose rows all stay where they were keeps its codes and its scale
        x = _blocks(torch.gather(_values(codes, scale, L), 1, kept[..., None].expand(-1, -1, D)))
        return torch.where(moved, _quantised(x), x).view(H, -1, D)[:, :m].transpose(0, 1).contiguous()

    return {"kept": kept.int(), "k": packed(s["k"], s["k_scale"]), "v": packed(s["v"], s["v_scale"]),
            "weight": torch.gather(w, 1, kept), "rows": m}


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    if case["op"] == "rope":
        return {"q": _rope(state["q"], state["pos"], case), "k": _rope(state["k"], state["pos"], case)}
    if case["op"] == "append":
        return {"k": _append(state, 0, state["new_k"]), "v": _append(state, 1, state["new_v"])}
    return _attend(state) if case["op"] == "attend" else _evict(state)


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------

def _library():
    here = os.path.join(os.getcwd(), "neon-runtime-beta-variation_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import neon_cuda

    return neon_cuda


def _cache(N, state, b):
    case = state["case"]
    return N.Kv8Cache(case["kv_heads"], case["dim"], b["k"].shape[1], b["k"], b["v"], b["k_scale"], b["v_scale"],
                      b["tail"], b["tail_block"], b["past"])


def _run_own(s):
    N = _library()
    case = s["case"]
    kind = {"f32": N.GGML_F32, "f16": N.GGML_F16, "bf16": N.GGML_BF16}.get(case.get("type"))
    H, D = case["kv_heads"], case["dim"]
    if case["op"] == "rope":
        if "spec" not in s:
            s["spec"] = N.Rope(case["rot"], half=case["half"], base=case["base"], scale=case["scale"],
                               yarn=1.0 if case["yarn"] else 0.0, orig_ctx=4096,
                               magnitude=0.1 * math.log(case["scale"]) + 1.0 if case["yarn"] else 1.0)
        q, k = torch.empty_like(s["q"]), torch.empty_like(s["k"])
        N.rope(s["spec"], s["pos"], case["n"], D, [(s["q"], q, case["heads"]), (s["k"], k, H)], type=kind,
               backward=case["back"])
        return {"q": q, "k": k}
    if "cache" not in s:  # a program keeps the cache and its workspace
        s["cache"] = _cache(N, s, s)
        if case["op"] == "attend":
            s["workspace"] = torch.empty(s["cache"].attention_workspace(case["heads"], case["n"]), dtype=torch.uint8,
                                         device="cuda")
        elif case["op"] == "evict":
            s["to"] = _cache(N, s, s["dst"])
            s["dst_weight"] = torch.zeros(H, s["dst"]["k"].shape[1], device="cuda")
    cache = s["cache"]
    if case["op"] == "append":
        n, r0 = case["n"], case["past"] % BLOCK
        cache.append(s["new_k"], s["new_v"], n, type=kind)
        k = torch.empty(r0 + n, H, D, device="cuda")
        v = torch.empty(r0 + n, H, D, device="cuda")
        cache.read(case["past"] - r0, r0 + n, k, v)
        return {"k": k, "v": v}
    if case["op"] == "attend":
        out = torch.empty_like(s["q"])
        w = s["weight"].clone() if case["weight"] else None
        cache.attention(s["q"], out, case["n"], case["heads"], s["workspace"], type=kind, weight=w)
        return {"out": out, "weight": w} if case["weight"] else {"out": out}
    m = min(case["past"], case["keep"])
    kept = torch.empty(H, case["keep"], dtype=torch.int32, device="cuda")
    cache.evict(s["to"], case["keep"], case["sink"], case["recent"], s["weight"], s["dst_weight"], kept)
    k = torch.empty(m, H, D, device="cuda")
    v = torch.empty(m, H, D, device="cuda")
    s["to"].read(0, m, k, v)
    return {"kept": kept[:, :m].contiguous(), "k": k, "v": v, "weight": s["dst_weight"][:, :m].contiguous(), "rows": m}


# ---------------------------------------------------------------------------
# what a pass cannot do without, and the definitions in 64 bits
# ---------------------------------------------------------------------------

def work(case):
    H, D = case["kv_heads"], case["dim"]
    size = {"f32": 4, "f16": 2, "bf16": 2}.get(case.get("type"), 4)
    if case["op"] == "rope":
        values = case["n"] * (case["heads"] + H) * D
        return {"bytes": 2 * size * values + 4 * case["n"], "flops": 3 * values}
    if case["op"] == "append":
        # new rows in, the block's earlier rows in, codes out, and the values read back
        values, before = 2 * case["n"] * H * D, 2 * (case["past"] % BLOCK) * H * D
        return {"bytes": size * values + 4 * before + 5 * (values + before), "flops": 4 * (values + before)}
    if case["op"] == "attend":
        n, past = case["n"], case["past"]
        rows = past + n
        pairs = case["heads"] * (n * past + n * (n + 1) // 2)
        moved = 2 * H * rows * D + 2 * 4 * H * ((rows + BLOCK - 1) // BLOCK) + 2 * size * n * case["heads"] * D
        if case["weight"]:
            moved += 8 * H * rows
        return {"bytes": moved, "flops": 4 * D * pairs}
    m = min(case["past"], case["keep"])
    return {"bytes": 4 * H * case["past"] + 2 * H * m * D * (1 + 1 + 4) + 8 * H * m, "flops": 4 * H * m * D}


def exact(case, seed):
    s = prepare(case, seed)
    H, D = case["kv_heads"], case["dim"]
    if case["op"] == "rope":
        rot = case["rot"]
        inv = []
        for i in range(rot // 2):
            f = case["base"] ** (-2.0 * i / rot)
            if case["yarn"]:
                # a pair that turns over 32 times in the first 4096 positions keeps its frequency, one that
                # turns less than once is stretched; between the two, by the pair's index
                first = math.floor(rot * math.log(4096 / (32 * 2 * math.pi)) / (2 * math.log(case["base"])))
                last = math.ceil(rot * math.log(4096 / (2 * math.pi)) / (2 * math.log(case["base"])))
                first, last = max(first, 0), min(last, rot - 1)
                part = min(1.0, max(0.0, (i - first) / max(last - first, 0.001)))
                f = f * (1 - part) + f / case["scale"] * part
            else:
                f = f / case["scale"]
            inv.append(f)
        size = 0.1 * math.log(case["scale"]) + 1.0 if case["yarn"] else 1.0
        z = torch.polar(torch.full((case["n"], rot // 2), size, dtype=torch.float64, device="cuda"),
                        s["pos"].double()[:, None] * torch.tensor(inv, dtype=torch.float64, device="cuda"))[:, None]
        z = z.conj() if case["back"] else z
        out = {}
        for name in ("q", "k"):
            x = s[name].double()
            r = x[..., :rot]
            pairs = torch.stack([r[..., :rot // 2], r[..., rot // 2:]], -1) if case["half"] else r.unflatten(-1, (-1, 2))
            y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * z)
            y = torch.cat([y[..., 0], y[..., 1]], -1) if case["half"] else y.flatten(-2)
            out[name] = torch.cat([y, x[..., rot:]], -1)
        return out

    def held(x):  # rows [n, D] of one head from a block's edge on, as 8 bits hold them
        y = torch.empty_like(x)
        for b in range(0, x.shape[0], BLOCK * 4096):
            part = x[b:b + BLOCK * 4096]
            pad = -part.shape[0] % BLOCK
            z = torch.cat([part, part.new_zeros(pad, D)]).view(-1, BLOCK * D)
            top = z.abs().max(1, keepdim=True).values
            step = (top / torch.full_like(top, 127.0)).float().double()  # a scale is an fp32 number
            step[top < TINY] = 0
            c = torch.round(z / step)
            c[(step == 0).expand_as(c)] = 0
            y[b:b + BLOCK * 4096] = (c * step).view(-1, D)[:part.shape[0]]
        return y

    if case["op"] == "append":
        r0, out = case["past"] % BLOCK, {}
        for i, name in enumerate(("k", "v")):
            heads = [held(torch.cat([s["tail"][i, 0, h, :r0].double(), s["new_" + name][:, h].double()])) for h in range(H)]
            out[name] = torch.stack(heads, 1)
        return out
    if case["op"] == "attend":
        n, past, group = case["n"], case["past"], case["heads"] // H
        rows = past + n
        out = torch.empty(n, case["heads"], D, dtype=torch.float64, device="cuda")
        w = s["weight"].double() if case["weight"] else None
        if w is not None:
            w[:, past:rows] = 0
        seen = torch.ones(n, rows, dtype=torch.bool, device="cuda").tril(past)
        for h in range(H):
            up = lambda x, sc: (x[h, :rows].view(rows, D).double() * sc[h].double().repeat_interleave(BLOCK)[:rows, None])  # noqa: E731
            k, v = up(s["k"], s["k_scale"]), up(s["v"], s["v_scale"])
            for j in range(h * group, (h + 1) * group):
                a = (s["q"][:, j].double() @ k.T) / math.sqrt(D)
                a = torch.softmax(a.masked_fill(~seen, -math.inf), dim=1)
                out[:, j] = a @ v
                if w is not None:
                    w[h, :rows] += a.sum(0)
        return {"out": out, "weight": w} if w is not None else {"out": out}
    L, keep, sink, recent = case["past"], case["keep"], case["sink"], case["recent"]
    m = min(L, keep)
    out = {"kept": None, "k": [], "v": [], "weight": [], "rows": None}
    for h in range(H):
        w = s["weight"][h, :L].cpu().numpy()
        if L > keep:
            middle = np.arange(sink, L - recent)
            best = middle[np.lexsort((middle, -w[middle]))][:keep - sink - recent]
            rows = np.concatenate([np.arange(sink), np.sort(best), np.arange(L - recent, L)])
        else:
            rows = np.arange(L)
        same = np.repeat(np.add.reduceat(rows != np.arange(m), np.arange(0, m, BLOCK)) == 0, BLOCK)[:m]
        at, same = torch.from_numpy(rows).cuda(), torch.from_numpy(same).cuda()
        for name in ("k", "v"):
            # a row's value is an fp32 number
            x = (s[name][h][at].double() * s[name + "_scale"][h][at // BLOCK].double()[:, None]).float().double()
            out[name].append(torch.where(same[:, None], x, held(x)))
        out["weight"].append(s["weight"][h][at].double())
    for name in ("k", "v"):
        out[name] = torch.stack(out[name], 1)
    out["weight"] = torch.stack(out["weight"])
    return out
