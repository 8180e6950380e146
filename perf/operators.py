"""What the attention-layer operators of a served batch are measured on: the cases, their inputs, the calls, and
the same operators in plain torch.

Three operators, the ones an attention layer needs when the requests of a batch differ from one another:

  lora    a linear layer with a low-rank adapter per row beside the shared weight
          Y = act(X W^T + bias + scale[a] (X A[a]^T) B[a]^T) + R,   a = row_adapter[row]  (negative: no adapter)
  cross   attention of padded queries over an encoder's states, with a key count, a query count and a key mask per
          request:  O = softmax(scale Q K^T over the valid keys) V  (no valid key: zero; rows behind the last
          query are left as they were)
  qk      RMS norm of every query and key head with the rotation by one to three position axes in the same pass

Sizes are those of the SD2.1 U-Net and its text encoder (C = 320 / 640 / 1280 at 64^2 / 32^2 / 16^2 tokens,
77-token prompts of width 1024, head dim 64) and generic ones.  How many rows, keys and queries a request has
follows from the case alone; every value comes from the seed.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one time-embedding projection row per request, each request with its own style adapter: pure latency
        dict(name="lora_time_rows", op="lora", M=8, per=1, K=1280, N=1280, r=16, L=8, dtype="f16", act="none", res=False),
        # single rows of many requests through the text MLP's up-projection, all adapters different
        dict(name="lora_rows_64", op="lora", M=64, per=1, K=1024, N=4096, r=32, L=64, dtype="bf16", act="gelu", res=False),
        # 13 prompts of 77 tokens: adapters change inside the row tiles, the last tile is ragged
        dict(name="lora_prompts", op="lora", M=1001, per=77, K=1024, N=4096, r=64, L=6, dtype="bf16", act="gelu", res=False),
        # fused q/k/v projection of 16 images at the 32x32 level
        dict(name="lora_qkv_32", op="lora", M=16384, per=1024, K=640, N=1920, r=16, L=8, dtype="f16", act="none", res=False),
        # output projection with its residual of 16 images at the 64x64 level: memory traffic
        dict(name="lora_out_64", op="lora", M=65536, per=4096, K=320, N=320, r=32, L=8, dtype="f16", act="none", res=True),
        # 16 images at the 64x64 level against prompts of 1 to 77 tokens
        dict(name="cross_prompts_64", op="cross", B=16, H=5, Hkv=5, D=64, Sq=4096, Skv=77, dtype="f16", mask=False, qlen=False),
        # odd sizes, holes in the key mask, a request without keys, padded queries
        dict(name="cross_odd_mask", op="cross", B=5, H=10, Hkv=10, D=64, Sq=333, Skv=231, dtype="f16", mask=True, qlen=True),
        # a long encoder sequence (a reference image's tokens) with shared key heads
        dict(name="cross_long", op="cross", B=2, H=8, Hkv=4, D=128, Sq=4096, Skv=8191, dtype="bf16", mask=False, qlen=False),
        # one query token per request over long encoder sequences: the keys' and values' bytes
        dict(name="cross_token", op="cross", B=16, H=16, Hkv=4, D=128, Sq=1, Skv=8192, dtype="bf16", mask=False, qlen=False),
        # two prompts, one position axis, halves rotated against each other: latency
        dict(name="qk_prompts", op="qk", T=154, P=77, Hq=16, Hk=16, D=64, axes="64", pairing="halves", dtype="f16", fused=True),
        # 16 images of 64x64 tokens, read in place from the fused q/k/v projection
        dict(name="qk_image_64", op="qk", T=65536, P=4096, Hq=5, Hk=5, D=64, axes="32,32", pairing="interleaved", dtype="f16", fused=True),
        # 16 frames of 30x45 tokens with time, height and width axes, fewer key heads than query heads
        dict(name="qk_video", op="qk", T=21600, P=21600, Hq=16, Hk=4, D=128, axes="16,56,56", pairing="interleaved", dtype="bf16", fused=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ranges; none costs more than the largest listed one of its operator."""
    op = rng.choice(("lora", "lora", "cross", "cross", "qk"))
    dtype = rng.choice(("f16", "bf16"))
    if op == "lora":
        K = 64 * _log(rng, 1, 64)
        N = 16 * _log(rng, 4, 256)
        top = min(65536.0, 20e9 / (K * N), 60e6 / (K + N))
        M = _log(rng, 1, max(2, top))
        per = 1 if M <= 128 else rng.choice((64, 77, 256, 1000, 4096))
        return dict(op=op, M=M, per=per, K=K, N=N, r=8 * rng.choice((1, 2, 2, 3, 4, 4, 8, 8, 16)), L=_log(rng, 1, 64),
                    dtype=dtype, act=rng.choice(("none", "none", "silu", "gelu")), res=rng.random() < 0.5)
    if op == "cross":
        D = rng.choice((64, 128))
        G = rng.choice((1, 1, 2, 3, 4, 8))
        Hkv = rng.randint(1, 10 if G == 1 else 4)
        B = rng.randint(1, 16)
        Skv = _log(rng, 1, 8192)
        per_key = B * Hkv * (2 * D)
        Skv = max(1, min(Skv, int(60e6 / per_key)))
        top = min(4096.0, 2 * 8 * 4096 * 8191 * 128 / (B * Hkv * G * Skv * D), 26e6 / (B * Hkv * G * D))
        Sq = 1 if rng.random() < 0.3 else _log(rng, 1, max(2, top))
        return dict(op=op, B=B, H=Hkv * G, Hkv=Hkv, D=D, Sq=Sq, Skv=Skv, dtype=dtype, mask=rng.random() < 0.4,
                    qlen=rng.random() < 0.3)
    D = rng.choice((64, 128))
    axes = rng.choice(("64", "32,32", "8,28,28", "16,24,24") if D == 64 else ("128", "64,64", "16,56,56", "32,48,48"))
    Hq = rng.randint(1, 24)
    Hk = rng.choice((0, 1, Hq, Hq))
    T = _log(rng, 1, min(65536.0, 40e6 / ((Hq + Hk) * D)))
    P = T if rng.random() < 0.5 else max(1, T // rng.randint(1, 8))
    return dict(op=op, T=T, P=P, Hq=Hq, Hk=Hk, D=D, axes=axes, pairing=rng.choice(("interleaved", "halves")), dtype=dtype,
                fused=rng.random() < 0.5)


# ---- what a case's requests look like -------------------------------------------------------------------------

def _adapter_rows(c):
    """row -> adapter: requests of `per` rows, every seventh request without an adapter."""
    n = -(-c["M"] // c["per"])
    ids = [-1 if i % 7 == 5 else (i * 5 + 2) % c["L"] for i in range(n)]
    return [ids[m // c["per"]] for m in range(c["M"])]


def _lengths(c, key, salt, empty):
    """One length per request in 1 .. c[key], the first of them full; with `empty` the last request has none."""
    r = random.Random("%s %d %d %d" % (salt, c["B"], c["Sq"], c["Skv"]))
    out = [c[key]] + [r.randint(max(1, c[key] // 8), c[key]) for _ in range(c["B"] - 1)]
    if empty and c["B"] > 1:
        out[-1] = 0
    return out


def _mask_rows(c):
    """[B][Skv] truth values: one key in five is masked out, at any place."""
    r = random.Random("mask %d %d" % (c["B"], c["Skv"]))
    return [[r.random() < 0.8 for _ in range(c["Skv"])] for _ in range(c["B"])]


def _sizes(c):
    kv = _lengths(c, "Skv", "kv", c["mask"])
    q = _lengths(c, "Sq", "q", False) if c["qlen"] else [c["Sq"]] * c["B"]
    return q, kv


def work(c):
    if c["op"] == "lora":
        M, K, N, r = c["M"], c["K"], c["N"], c["r"]
        rows = _adapter_rows(c)
        used, with_adapter = len(set(a for a in rows if a >= 0)), sum(a >= 0 for a in rows)
        n = M * K + N * K + M * N * (2 if c["res"] else 1) + used * r * (K + N)
        return {"bytes": 2 * n + 4 * (M + N + c["L"]), "flops": 2 * M * N * K + 2 * with_adapter * r * (K + N)}
    if c["op"] == "cross":
        q, kv = _sizes(c)
        keys = [sum(m[:n]) for m, n in zip(_mask_rows(c), kv)] if c["mask"] else kv
        n = sum(2 * a * c["H"] * c["D"] + 2 * k * c["Hkv"] * c["D"] for a, k in zip(q, keys))
        return {"bytes": 2 * n + 8 * c["B"] + (c["B"] * c["Skv"] if c["mask"] else 0),
                "flops": 4 * sum(a * k for a, k in zip(q, keys)) * c["H"] * c["D"]}
    n = c["T"] * (c["Hq"] + c["Hk"]) * c["D"]
    return {"bytes": 4 * n + 4 * c["P"] * (c["axes"].count(",") + 1) + 8 * c["D"], "flops": 8 * n}


# ---- inputs ---------------------------------------------------------------------------------------------------

def prepare(c, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    dt = _DT[c["dtype"]]

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(shape, generator=g, device=dev) * scale).to(dtype)

    s = {"case": c}
    if c["op"] == "lora":
        M, K, N, r, L = c["M"], c["K"], c["N"], c["r"], c["L"]
        s["x"] = normal(M, K)
        s["w"] = normal(N, K, scale=K ** -0.5)
        s["a"] = normal(L, r, K, scale=K ** -0.5)
        s["b"] = normal(L, N, r, scale=0.5 * r ** -0.5)
        s["scale"] = 0.5 + torch.rand(L, generator=g, device=dev)
        s["rows"] = torch.tensor(_adapter_rows(c), dtype=torch.int32, device=dev)
        s["bias"] = normal(N, scale=0.2, dtype=torch.float32)
        s["res"] = normal(M, N) if c["res"] else None
        s["out"] = torch.empty(M, N, dtype=dt, device=dev)
    elif c["op"] == "cross":
        B, Sq, Skv, H, Hkv, D = (c[k] for k in ("B", "Sq", "Skv", "H", "Hkv", "D"))
        q, kv = _sizes(c)
        s["q"] = normal(B, Sq, H, D)
        both = normal(B, Skv, 2, Hkv, D)  # keys and values of one fused projection
        s["k"], s["v"] = both[:, :, 0], both[:, :, 1]
        s["kv_len"] = torch.tensor(kv, dtype=torch.int32, device=dev)
        s["q_len"] = torch.tensor(q, dtype=torch.int32, device=dev) if c["qlen"] else None
        s["mask"] = torch.tensor(_mask_rows(c), dtype=torch.uint8, device=dev) if c["mask"] else None
        s["out"] = torch.zeros(B, Sq, H, D, dtype=dt, device=dev)
    else:
        T, P, Hq, Hk, D = (c[k] for k in ("T", "P", "Hq", "Hk", "D"))
        if c["fused"]:  # rows of the fused projection: q heads, k heads, as many v heads
            x = normal(T, Hq + 2 * Hk, D, scale=2.0)
            s["q"], s["k"] = x[:, :Hq], x[:, Hq:Hq + Hk] if Hk else None
        else:
            s["q"] = normal(T, Hq, D, scale=2.0)
            s["k"] = normal(T, Hk, D, scale=2.0) if Hk else None
        s["wq"] = 1 + normal(D, scale=0.1, dtype=torch.float32)
        s["wk"] = 1 + normal(D, scale=0.1, dtype=torch.float32)
        s["axes"] = tuple(int(a) for a in c["axes"].split(","))
        # token grid: the first axis runs slowest, as frames, rows and columns do; odd seeds start far into a sequence
        side = [max(1, round(P ** (1.0 / len(s["axes"]))))] * len(s["axes"])
        p = torch.arange(P, device=dev)
        cols = [p // side[1] // side[2] if len(side) == 3 else p // side[-1] if len(side) == 2 else p]
        cols += [p // side[2] % side[1]] if len(side) == 3 else []
        cols += [p % side[-1]] if len(side) > 1 else []
        s["pos"] = (torch.stack(cols, 1) + (100003 if seed % 2 else 0)).to(torch.int32).contiguous()
        s["q_out"] = torch.empty(T, Hq, D, dtype=dt, device=dev)
        s["k_out"] = torch.empty(T, Hk, D, dtype=dt, device=dev) if Hk else None
    return s


# ---- one pass -------------------------------------------------------------------------------------------------

_ctx = None


def _layers():
    """The framework's layers module and a context on the current device (its directory name has a hyphen)."""
    global _ctx
    import sys
    if "draw_instant_b200" not in sys.modules:
        import importlib.util
        spec = importlib.util.spec_from_file_location("draw_instant_b200", "draw-instant_b200/__init__.py",
                                                      submodule_search_locations=["draw-instant_b200"])
        sys.modules["draw_instant_b200"] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules["draw_instant_b200"])
    from draw_instant_b200 import default_context, layers
    if _ctx is None:
        _ctx = default_context(torch.cuda.current_device())
    return layers, _ctx


def run(s):
    op = s["case"]["op"]
    if own:
        layers, ctx = _layers()
        if op == "lora":
            return layers.linear_lora(ctx, s["x"], s["w"], s["a"], s["b"], s["scale"], s["rows"], bias=s["bias"],
                                      residual=s["res"], act=s["case"]["act"], out=s["out"])
        if op == "cross":
            return layers.cross_attention(ctx, s["q"], s["k"], s["v"], kv_len=s["kv_len"], q_len=s["q_len"],
                                          key_mask=s["mask"], out=s["out"])
        return layers.qk_norm_rope(ctx, s["q"], s["k"], q_weight=s["wq"], k_weight=s["wk"], eps=1e-6,
                                   positions=s["pos"], axis_dims=s["axes"], theta=10000.0,
                                   pairing=s["case"]["pairing"], q_out=s["q_out"], k_out=s["k_out"])
    return {"lora": _plain_lora, "cross": _plain_cross, "qk": _plain_qk}[op](s)


def _plain_lora(s):
    """Every adapter at every row, and the rows' own ones kept."""
    c, x = s["case"], s["x"].float()
    L, r, K = s["a"].shape
    t = (x @ s["a"].float().reshape(L * r, K).T).reshape(-1, L, r)
    mine = s["rows"].long()[:, None] == torch.arange(L, device=x.device)
    t = torch.where(mine[:, :, None], t * s["scale"][:, None], torch.zeros((), device=x.device))
    y = x @ s["w"].float().T + s["bias"]
    y = y + t.reshape(-1, L * r) @ s["b"].float().permute(0, 2, 1).reshape(L * r, -1)
    if c["act"] == "silu":
        y = y / (1 + torch.exp(-y))
    elif c["act"] == "gelu":
        y = 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    if s["res"] is not None:
        y = y + s["res"].float()
    return y.to(s["x"].dtype)


def _plain_cross(s):
    c, q = s["case"], s["q"].float()
    B, Sq, H, D = q.shape
    Skv, Hkv = s["k"].shape[1:3]
    k, v = s["k"].float(), s["v"].float()
    scores = torch.einsum("bihgd,bjhd->bhgij", q.reshape(B, Sq, Hkv, H // Hkv, D), k) * D ** -0.5
    ok = torch.arange(Skv, device=q.device) < s["kv_len"][:, None]
    if s["mask"] is not None:
        ok = ok & (s["mask"] != 0)
    ok = ok[:, None, None, None, :]
    scores = torch.where(ok, scores, torch.full((), -math.inf, device=q.device))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1)
    o = torch.einsum("bhgij,bjhd->bhgid", p, v) / torch.where(total > 0, total, torch.ones_like(total))[..., None]
    o = o.permute(0, 3, 1, 2, 4).reshape(B, Sq, H, D).to(s["q"].dtype)
    if s["q_len"] is None:
        return o
    return torch.where((torch.arange(Sq, device=q.device) < s["q_len"][:, None])[:, :, None, None], o, s["out"])


def _plain_rotate(s, x, w):
    c, D = s["case"], x.shape[-1]
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
    axis, index, width = (torch.tensor(v, device=x.device) for v in zip(*[(a, j, d) for a, d in enumerate(s["axes"]) for j in range(d // 2)]))
    freq = torch.exp(-math.log(10000.0) * (2 * index).double() / width.double())
    angle = s["pos"].double()[:, axis] * freq
    angle = angle.repeat(-(-x.shape[0] // angle.shape[0]), 1)[:x.shape[0], None, :]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    if c["pairing"] == "halves":
        lo, hi = x[..., :D // 2], x[..., D // 2:]
        y = torch.cat([lo * cos - hi * sin, lo * sin + hi * cos], -1)
    else:
        lo, hi = x[..., 0::2], x[..., 1::2]
        y = torch.stack([lo * cos - hi * sin, lo * sin + hi * cos], -1).flatten(-2)
    return y.to(s["q"].dtype)


def _plain_qk(s):
    if s["k"] is None:
        return _plain_rotate(s, s["q"], s["wq"])
    return _plain_rotate(s, s["q"], s["wq"]), _plain_rotate(s, s["k"], s["wk"])


# ---- the definition in 64 bits --------------------------------------------------------------------------------

def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "lora":
        x, w = s["x"].double(), s["w"].double()
        y = x @ w.mT + s["bias"].double()
        rows = s["rows"].cpu()
        for a in sorted(set(rows.tolist())):
            if a >= 0:
                at = (rows == a).nonzero()[:, 0].to(x.device)
                y[at] += s["scale"][a].double() * ((x[at] @ s["a"][a].double().mT) @ s["b"][a].double().mT)
        if c["act"] == "silu":
            y = y * torch.sigmoid(y)
        elif c["act"] == "gelu":
            y = y * (torch.special.erfc(-y / math.sqrt(2.0)) / 2)
        return y + s["res"].double() if s["res"] is not None else y
    if c["op"] == "cross":
        out = s["out"].double()
        group = c["H"] // c["Hkv"]
        queries, keys = _sizes(c)
        for b in range(c["B"]):
            at = torch.arange(keys[b], device=out.device)
            if s["mask"] is not None:
                at = at[s["mask"][b, :keys[b]] != 0]
            for h in range(c["H"]):
                q = s["q"][b, :queries[b], h].double()
                k, v = s["k"][b, at, h // group].double(), s["v"][b, at, h // group].double()
                out[b, :queries[b], h] = torch.softmax(q @ k.mT / math.sqrt(c["D"]), -1) @ v if len(at) else 0.0
        return out
    outs = []
    for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
        if x is None:
            continue
        x = x.double()
        x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / c["D"] + 1e-6) * w.double()
        z, first = [], 0
        pos = s["pos"][torch.arange(c["T"], device=x.device) % c["P"]].double()
        pairs = torch.view_as_complex(x.unflatten(-1, (2, -1)).transpose(-1, -2).contiguous() if c["pairing"] == "halves"
                                      else x.unflatten(-1, (-1, 2)).contiguous())
        for axis, d in enumerate(s["axes"]):
            turn = pos[:, axis, None] / 10000.0 ** (torch.arange(0, d, 2, device=x.device).double() / d)
            z.append(pairs[..., first:first + d // 2] * torch.polar(torch.ones_like(turn), turn)[:, None])
            first += d // 2
        y = torch.view_as_real(torch.cat(z, -1))
        outs.append((y.transpose(-1, -2) if c["pairing"] == "halves" else y).flatten(-2).contiguous())
    return tuple(outs) if len(outs) > 1 else outs[0]
