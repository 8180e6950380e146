"""The layers module (per-row adapters, head norms with rotation, attention over encoder states) against plain 64-bit
formulas on the same 16-bit inputs.

Tolerances follow from the arithmetic, elementwise.  h is half a step of the output type (2^-11 fp16, 2^-8 bf16), u = 2^-23
one fp32 step:
  lora   one rounding of the result, h |y|; the fp32 sums of K and r products, accumulated in chunks of 16, drift by at
         most (K / 16 + r / 16 + 32) u S with S the sum of the absolute terms; the adapter's inner value enters the second
         product as two 16-bit parts, 2^-16 of the sum of |t b| (and 2^-25 absolute per part in fp16).  The activations'
         slope is at most 1.13.
  cross  h |o| for the result and h sum(p |v|) for the 16-bit probabilities; a score is off by at most D u sum(|q k|) scale
         and the exponential by 2^-21, both relative for p and for the sum; in fp16 a probability below 2^-14 of the largest
         is off by up to 2^-25 of it.
  qk     h |y| and a few fp32 steps of the pair's length: 16 u (|x| w / rms summed over the pair).
fp16 results below 2^-14 round to multiples of 2^-24: half of that is added throughout."""
from __future__ import annotations

import importlib
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16}
H = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
U = 2.0 ** -23
TINY = 2.0 ** -25


@pytest.fixture(scope="module")
def layers(dib):
    return importlib.import_module("draw_instant_b200.layers")


def normal(gen, *shape, dt=torch.float16, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dt)


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def check(got, ref, tol, what=""):
    got = got.double()
    bad = ~((got - ref).abs() <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} outside, first at {bad.nonzero()[0].tolist()}: "
                           f"got {got[bad][0].item()}, want {ref[bad][0].item()} +- {tol[bad][0].item()}")


# ---- linear_lora ----------------------------------------------------------------------------------------------

def lora_case(seed, M, K, N, r, L, dt, bias=True, res=False, rows=None):
    g = gen(seed)
    s = dict(x=normal(g, M, K, dt=dt), w=normal(g, N, K, dt=dt, scale=K ** -0.5),
             a=normal(g, L, r, K, dt=dt, scale=K ** -0.5), b=normal(g, L, N, r, dt=dt, scale=r ** -0.5),
             scale=0.5 + torch.rand(L, generator=g, device="cuda"))
    s["row_adapter"] = torch.randint(-1, L, (M,), generator=g, device="cuda").int() if rows is None else torch.tensor(
        rows, dtype=torch.int32, device="cuda")
    s["bias"] = normal(g, N, dt=torch.float32) if bias else None
    s["residual"] = normal(g, M, N, dt=dt) if res else None
    return s


def lora_ref(s, act="none"):
    """(result, tolerance) in 64 bits."""
    x, w, a, b = (s[k].double() for k in ("x", "w", "a", "b"))
    dt, K, r = s["x"].dtype, x.shape[1], a.shape[1]
    rows = s["row_adapter"].long()
    rows = torch.where(rows >= a.shape[0], torch.full_like(rows, -1), rows)
    y, mag, inner = x @ w.T, x.abs() @ w.abs().T, torch.zeros(len(x), len(w), device="cuda", dtype=torch.float64)
    for i in rows.unique().tolist():
        if i < 0:
            continue
        at = rows == i
        f = s["scale"][i].double()
        t, tm = f * (x[at] @ a[i].T), f * (x[at].abs() @ a[i].abs().T)
        y[at] += t @ b[i].T
        mag[at] += tm @ b[i].abs().T
        inner[at] += t.abs() @ b[i].abs().T * 2.0 ** -16 + (2 * TINY * b[i].abs().sum(1) if dt == torch.float16 else 0)
    if s["bias"] is not None:
        y = y + s["bias"].double()
        mag = mag + s["bias"].double().abs()
    slack = (K / 16 + r / 16 + 32) * U * mag + inner
    if act == "silu":
        y, slack = y * torch.sigmoid(y), 1.13 * slack + 8 * U * y.abs()
    elif act == "gelu":
        slack = 1.13 * slack + (2e-7 + 8 * U) * y.abs()
        y = y * torch.special.erfc(-y / math.sqrt(2)) / 2
    if s["residual"] is not None:
        y = y + s["residual"].double()
        slack = slack + U * s["residual"].double().abs()
    return y, H[dt] * y.abs() + (1 + H[dt]) * slack + TINY


LORA = [  # M, K, N, r, L
    (1, 64, 16, 8, 1), (1, 1280, 1280, 16, 4), (2, 320, 48, 24, 3), (7, 1024, 4096, 64, 9), (8, 1280, 320, 16, 8),
    (16, 640, 640, 128, 5), (33, 192, 176, 40, 33), (64, 1024, 1024, 32, 64), (65, 640, 208, 16, 3),
    (127, 320, 320, 8, 20), (128, 320, 320, 64, 2), (129, 1280, 336, 128, 40), (300, 704, 960, 48, 7),
    (9, 64, 16, 128, 2), (12, 640, 1536, 16, 4), (13, 640, 1552, 16, 4), (25, 320, 1568, 64, 1), (32, 128, 384, 8, 5),
    (44, 1408, 192, 128, 3), (106, 64, 256, 64, 2), (128, 64, 4096, 128, 7), (64, 320, 4784, 64, 5), (33, 128, 2400, 24, 33),
    (1001, 1024, 4096, 64, 6), (2048, 320, 640, 104, 16), (4097, 128, 32, 16, 2), (20000, 320, 320, 32, 8)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("M,K,N,r,L", LORA)
def test_lora_rows_in_any_order(ctx, layers, M, K, N, r, L, dtype):
    """Every row with an adapter of its own choosing, neighbours mostly different."""
    s = lora_case(M * 31 + N, M, K, N, r, L, DT[dtype], bias=M % 2 == 0, res=M % 3 == 0)
    act = ("none", "silu", "gelu")[(M + r) % 3]
    got = layers.linear_lora(ctx, **s, act=act)
    check(got, *lora_ref(s, act))
    assert ctx.fault() == 0


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("M,per,K,N,r,L", [(1001, 77, 1024, 1024, 16, 6), (2048, 64, 640, 1920, 32, 30), (8192, 1024, 640, 640, 16, 8),
                                           (700, 100, 320, 320, 128, 3), (513, 256, 1280, 1280, 64, 4)])
def test_lora_requests(ctx, layers, M, per, K, N, r, L, dtype):
    """Whole requests with one adapter each, some without."""
    ids = [-1 if i % 5 == 3 else (i * 3) % L for i in range(-(-M // per))]
    s = lora_case(M + per, M, K, N, r, L, DT[dtype], res=True, rows=[ids[m // per] for m in range(M)])
    check(layers.linear_lora(ctx, **s), *lora_ref(s))
    assert ctx.fault() == 0


@pytest.mark.parametrize("M", [5, 200])
def test_lora_without_any_adapter_is_the_linear_layer(ctx, dib, layers, M):
    s = lora_case(3, M, 320, 320, 16, 2, torch.float16, rows=[-1] * M)
    s["a"].fill_(float("nan"))  # never used: must not reach the result
    s["b"].fill_(float("inf"))
    got = layers.linear_lora(ctx, **s)
    s["a"].zero_(), s["b"].zero_()
    check(got, *lora_ref(s))


@pytest.mark.parametrize("M", [6, 150, 1000])
def test_lora_unused_adapters_and_other_rows_do_not_mix(ctx, layers, M):
    """An adapter of NaN and infinities shows only in the rows that name it."""
    s = lora_case(5, M, 640, 320, 32, 4, torch.bfloat16)
    mine = s["row_adapter"] == 2
    s["a"][2], s["b"][2] = float("nan"), float("inf")
    got = layers.linear_lora(ctx, **s)
    assert torch.isnan(got[mine]).all()
    s["a"][2], s["b"][2] = 0, 0
    ref, tol = lora_ref(s)
    check(got[~mine], ref[~mine], tol[~mine])


@pytest.mark.parametrize("M", [6, 150])
def test_lora_nan_rows_stay_in_their_rows(ctx, layers, M):
    s = lora_case(6, M, 320, 320, 16, 4, torch.float16)
    s["x"][M // 2] = float("nan")
    s["x"][0, 0] = float("inf")
    got = layers.linear_lora(ctx, **s)
    keep = torch.ones(M, dtype=torch.bool, device="cuda")
    keep[M // 2] = keep[0] = False
    assert torch.isnan(got[M // 2]).all() and not torch.isfinite(got[0]).any()
    s["x"][M // 2] = 0
    s["x"][0, 0] = 0
    ref, tol = lora_ref(s)
    check(got[keep], ref[keep], tol[keep])


@pytest.mark.parametrize("M", [9, 140])
def test_lora_index_past_the_last_adapter_is_flagged(ctx, layers, M):
    s = lora_case(7, M, 320, 64, 16, 3, torch.float16)
    s["row_adapter"][M - 1] = 3
    s["row_adapter"][0] = 2 ** 31 - 1
    got = layers.linear_lora(ctx, **s)
    assert ctx.fault() == 16
    ctx.clear_fault()
    check(got, *lora_ref(s))


@pytest.mark.parametrize("M", [10, 300])
def test_lora_strided_rows_in_place_residual_and_surroundings(ctx, layers, M):
    """x is a slice of a wider buffer, the residual is the output, and what lies around the output stays."""
    dt = torch.float16
    s = lora_case(8, M, 320, 336, 16, 3, dt, res=True)
    wide = torch.full((M, 400), 7.0, dtype=dt, device="cuda")
    wide[:, 40:360] = s["x"]
    hold = torch.full((M + 2, 400), 5.0, dtype=dt, device="cuda")
    hold[1:-1, 32:368] = s["residual"]
    ref = lora_ref(s)
    y = hold[1:-1, 32:368]
    got = layers.linear_lora(ctx, **{**s, "x": wide[:, 40:360], "residual": y}, out=y)
    assert got.data_ptr() == y.data_ptr()
    check(got, *ref)
    around = hold.clone()
    around[1:-1, 32:368] = 5.0
    assert (around == 5.0).all()


@pytest.mark.parametrize("M", [40, 300])
@pytest.mark.parametrize("ld,at", [(344, 0), (352, 8), (352, 16)])
def test_lora_rows_on_16_bytes(ctx, layers, M, ld, at):
    """Output and residual rows that start on 16 bytes, but not on 32."""
    s = lora_case(10, M, 320, 336, 16, 3, torch.bfloat16, res=True)
    hold, held = torch.zeros(M, ld, dtype=torch.bfloat16, device="cuda"), torch.zeros(M, ld, dtype=torch.bfloat16, device="cuda")
    at = min(at, ld - 336)
    held[:, at:at + 336] = s["residual"]
    ref = lora_ref(s, "silu")
    check(layers.linear_lora(ctx, **{**s, "residual": held[:, at:at + 336]}, act="silu", out=hold[:, at:at + 336]), *ref)
    assert (hold[:, :at] == 0).all() and (hold[:, at + 336:] == 0).all()


@pytest.mark.parametrize("M", [12, 1000])
def test_lora_repeats_bit_for_bit(ctx, layers, M):
    s = lora_case(9, M, 1280, 640, 32, 6, torch.bfloat16, res=True)
    first = layers.linear_lora(ctx, **s, act="silu")
    for _ in range(3):
        assert torch.equal(layers.linear_lora(ctx, **s, act="silu"), first)


@pytest.mark.parametrize("M,per,K,N,r,L", [(1001, 77, 640, 1280, 64, 6), (3000, 50, 320, 320, 32, 9), (70, 1, 640, 640, 16, 70)])
def test_lora_back_to_back(ctx, layers, M, per, K, N, r, L):
    """Thirty calls queued at once: every one gives the same bits, and the right ones."""
    s = lora_case(M, M, K, N, r, L, torch.float16, res=True, rows=[(m // per * 5) % (L + 1) - 1 for m in range(M)])
    outs = [layers.linear_lora(ctx, **s, act="gelu") for _ in range(30)]
    check(outs[0], *lora_ref(s, "gelu"))
    for o in outs[1:]:
        assert torch.equal(o, outs[0])


def test_lora_c_entry_refusals(ctx, dib):
    import ctypes
    L, s = dib.lib(), lora_case(1, 4, 64, 32, 8, 2, torch.float16)
    y = torch.empty(4, 32, dtype=torch.float16, device="cuda")
    ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")

    def call(**k):
        c = dict(M=4, N=32, K=64, r=8, L=2, ldx=64, ldr=0, ldy=32, act=0)
        v = dict(dtype=1, cfg=None, X=s["x"].data_ptr(), W=s["w"].data_ptr(), A=s["a"].data_ptr(), B=s["b"].data_ptr(),
                 scale=s["scale"].data_ptr(), rows=s["row_adapter"].data_ptr(), bias=None, R=None, Y=y.data_ptr(), ws=ws.data_ptr(),
                 n=ws.numel())
        for key, val in k.items():
            (c if key in c else v)[key] = val
        v["cfg"] = (ctypes.c_longlong * 9)(*c.values())
        return L.di_linear_lora(ctx.h, *v.values())

    assert call() == 0
    for bad in (dict(dtype=0), dict(M=0), dict(M=-1), dict(M=1 << 40), dict(N=0), dict(L=0), dict(X=None), dict(A=None), dict(rows=None),
                dict(ldx=56), dict(ldx=68), dict(ldy=24), dict(ldy=36), dict(X=s["x"].data_ptr() + 2), dict(Y=y.data_ptr() + 8),
                dict(act=3), dict(act=-1), dict(R=y.data_ptr(), ldr=0)):
        assert call(**bad) == dib.DI_EINVAL, bad
    for bad in (dict(K=32), dict(K=96), dict(N=24), dict(r=12), dict(r=0), dict(r=136)):
        assert call(**bad) == dib.DI_EUNSUPPORTED, bad
    for M in (4, 64, 500):  # scratch that is missing, too small or misaligned (M rows need not exist: nothing is launched)
        need = L.di_linear_lora_workspace(ctx.h, (ctypes.c_longlong * 9)(M, 32, 64, 8, 2, 64, 0, 32, 0))
        if need:
            for bad in (dict(ws=None), dict(n=need - 1), dict(ws=ws.data_ptr() + 8)):
                assert call(M=M, **bad) == dib.DI_EINVAL, bad


# ---- qk_norm_rope ---------------------------------------------------------------------------------------------

def qk_ref(x, w, eps, pos, dims, theta, pairing):
    """(result, tolerance) of one of the two tensors in 64 bits."""
    T, _, D = x.shape
    f = x.double()
    if w is not None:
        f = f / torch.sqrt(f.pow(2).mean(-1, keepdim=True) + eps) * w.double()
    pair = (lambda t: (t[..., :D // 2], t[..., D // 2:])) if pairing == "halves" else (lambda t: (t[..., 0::2], t[..., 1::2]))
    lo, hi = pair(f)
    if pos is not None:
        at = torch.arange(T, device="cuda") % pos.shape[0]
        ang = torch.cat([pos[at, a, None].double() * theta ** (-torch.arange(0, d, 2, device="cuda").double() / d)
                         for a, d in enumerate(dims)], 1)[:, None]
        c, s = torch.cos(ang), torch.sin(ang)
        size = lo.abs() + hi.abs()
        lo, hi = lo * c - hi * s, lo * s + hi * c
    else:
        size = torch.maximum(lo.abs(), hi.abs())
    if pairing == "halves":
        y, size = torch.cat([lo, hi], -1), torch.cat([size, size], -1)
    else:
        y, size = torch.stack([lo, hi], -1).flatten(-2), torch.stack([size, size], -1).flatten(-2)
    return y, H[x.dtype] * y.abs() + 16 * U * size + TINY


def grid_positions(g, P, n, far):
    pos = torch.randint(0, 64, (P, n), generator=g, device="cuda")
    if far:
        pos = pos + torch.randint(-2 ** 31, 2 ** 31 - 64, (P, n), generator=g, device="cuda")
    return pos.int()


QK = [  # T, Hq, Hk, D, dims
    (1, 1, 0, 64, (64,)), (1, 3, 1, 128, (16, 56, 56)), (154, 16, 16, 64, (64,)), (33, 5, 5, 64, (32, 32)),
    (333, 7, 2, 128, (64, 64)), (4096, 10, 10, 64, (8, 28, 28)), (777, 24, 3, 128, (128,)), (30000, 2, 1, 64, (2, 60, 2))]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("pairing", ["interleaved", "halves"])
@pytest.mark.parametrize("T,Hq,Hk,D,dims", QK)
def test_qk(ctx, layers, T, Hq, Hk, D, dims, pairing, dtype):
    g = gen(T + Hq)
    dt = DT[dtype]
    q, k = normal(g, T, Hq, D, dt=dt, scale=3.0), normal(g, T, Hk, D, dt=dt, scale=0.1) if Hk else None
    wq, wk = 1 + normal(g, D, dt=torch.float32, scale=0.3), 1 + normal(g, D, dt=torch.float32, scale=0.3)
    P = max(1, T // 3)
    pos = grid_positions(g, P, len(dims), far=T % 2 == 1)
    got = layers.qk_norm_rope(ctx, q, k, q_weight=wq, k_weight=wk, eps=1e-5, positions=pos, axis_dims=dims, theta=500.0,
                              pairing=pairing)
    for y, x, w in zip(got if Hk else (got,), (q, k), (wq, wk)):
        check(y, *qk_ref(x, w, 1e-5, pos, dims, 500.0, pairing))


@pytest.mark.parametrize("pairing", ["interleaved", "halves"])
def test_qk_norm_or_rotation_alone(ctx, layers, pairing):
    g = gen(2)
    q, k = normal(g, 50, 3, 64), normal(g, 50, 2, 64)
    w = 1 + normal(g, 64, dt=torch.float32, scale=0.3)
    pos = grid_positions(g, 50, 1, False)
    y, z = layers.qk_norm_rope(ctx, q, k, k_weight=w, pairing=pairing)  # a norm for k only, no rotation
    assert torch.equal(y, q)
    check(z, *qk_ref(k, w, 1e-6, None, (), 1.0, pairing))
    y = layers.qk_norm_rope(ctx, q, positions=pos, axis_dims=(64,), pairing=pairing)
    check(y, *qk_ref(q, None, 0, pos, (64,), 10000.0, pairing))


@pytest.mark.parametrize("pairing", ["interleaved", "halves"])
@pytest.mark.parametrize("D,dims", [(64, (32, 32)), (128, (16, 56, 56))])
def test_qk_in_place_in_a_fused_projection(ctx, layers, D, dims, pairing):
    """q and k are rotated where they lie; the values beside them stay."""
    g = gen(4)
    x = normal(g, 1000, 3 * 5, D, dt=torch.bfloat16)
    before = x.clone()
    w = 1 + normal(g, D, dt=torch.float32, scale=0.3)
    pos = grid_positions(g, 250, len(dims), False)
    q, k = x[:, :5], x[:, 5:10]
    layers.qk_norm_rope(ctx, q, k, q_weight=w, k_weight=w, positions=pos, axis_dims=dims, pairing=pairing, q_out=q, k_out=k)
    check(q, *qk_ref(before[:, :5], w, 1e-6, pos, dims, 10000.0, pairing))
    check(k, *qk_ref(before[:, 5:10], w, 1e-6, pos, dims, 10000.0, pairing))
    assert torch.equal(x[:, 10:], before[:, 10:])


def test_qk_special_values_stay_in_their_heads(ctx, layers):
    q = torch.ones(6, 4, 64, dtype=torch.float16, device="cuda")
    q[1, 2, 5], q[3, 0, 0], q[4, 1] = float("nan"), float("inf"), 0.0
    w = torch.ones(64, device="cuda")
    y = layers.qk_norm_rope(ctx, q, q_weight=w, eps=1e-6)
    bad = torch.isnan(y).any(-1)
    assert bad.nonzero().tolist() == [[1, 2], [3, 0]] and (y[4, 1] == 0).all()
    assert (y[0] == 1).all()


def test_qk_c_entry_refusals(ctx, dib):
    import ctypes
    L = dib.lib()
    q = torch.zeros(4, 2, 64, dtype=torch.float16, device="cuda")
    pos = torch.zeros(4, 2, dtype=torch.int32, device="cuda")

    def call(dims=(32, 32), **k):
        c = dict(T=4, Hq=2, Hk=0, D=64, ldq=128, ldk=0, ldqo=128, ldko=0, P=4, pairing=0, n=len(dims))
        v = dict(dtype=1, cfg=None, eps=1e-6, theta=1e4, Q=q.data_ptr(), K=None, wq=None, wk=None, pos=pos.data_ptr(),
                 Qo=q.data_ptr(), Ko=None)
        for key, val in k.items():
            (c if key in c else v)[key] = val
        v["cfg"] = (ctypes.c_longlong * 16)(*c.values(), *dims)
        return L.di_qk_norm_rope(ctx.h, *v.values())

    assert call() == 0
    for bad in (dict(dtype=0), dict(T=0), dict(T=-4), dict(Hq=0), dict(Q=None), dict(Hk=1), dict(K=q.data_ptr()), dict(ldq=64),
                dict(ldq=132), dict(Q=q.data_ptr() + 2), dict(dims=(32, 16)), dict(dims=(33, 31)), dict(dims=(32, 32, -2)),
                dict(dims=()), dict(dims=(16, 16, 16, 16)), dict(P=0), dict(theta=0.0), dict(pairing=2), dict(eps=-1.0),
                dict(eps=float("nan"))):
        assert call(**bad) == dib.DI_EINVAL, bad
    assert call(D=96) == dib.DI_EUNSUPPORTED


# ---- cross_attention ------------------------------------------------------------------------------------------

def cross_ref(q, k, v, kv_len=None, q_len=None, key_mask=None, scale=None, out=None):
    """(result, tolerance) in 64 bits; rows behind q_len as in `out`."""
    B, Sq, Hq, D = q.shape
    Skv, Hkv = k.shape[1:3]
    dt = q.dtype
    scale = D ** -0.5 if scale is None else scale
    ref = torch.zeros(B, Sq, Hq, D, dtype=torch.float64, device="cuda") if out is None else out.double().clone()
    tol = torch.zeros_like(ref)
    for b in range(B):
        n = Skv if kv_len is None else min(max(int(kv_len[b]), 0), Skv)
        m = Sq if q_len is None else min(max(int(q_len[b]), 0), Sq)
        at = torch.arange(n, device="cuda")
        if key_mask is not None:
            at = at[key_mask[b, :n] != 0]
        for h in range(Hq):
            if len(at) == 0:
                ref[b, :m, h] = 0
                continue
            qq, kk, vv = q[b, :m, h].double(), k[b, at, h // (Hq // Hkv)].double(), v[b, at, h // (Hq // Hkv)].double()
            s = qq @ kk.T * scale
            p = torch.softmax(s, -1)
            o, ov = p @ vv, p @ vv.abs()
            off = D * U * scale * (qq.abs() @ kk.abs().T).amax(-1, keepdim=True) + 2.0 ** -21 + len(at) / 16 * U
            ref[b, :m, h] = o
            t = H[dt] * o.abs() + (H[dt] + 2 * off) * ov + TINY
            if dt == torch.float16:
                t = t + len(at) * TINY * p.amax(-1, keepdim=True) * vv.abs().amax()
            tol[b, :m, h] = t
    return ref, tol


CROSS = [  # B, Sq, Skv, H, Hkv, D
    (1, 1, 1, 1, 1, 64), (1, 1, 1, 1, 1, 128), (2, 1, 77, 5, 5, 64), (3, 1, 1000, 8, 1, 128), (2, 3, 4097, 6, 2, 64),
    (2, 64, 64, 2, 2, 64), (2, 65, 63, 3, 3, 128), (2, 127, 128, 4, 4, 64), (1, 129, 129, 4, 2, 128), (2, 333, 231, 10, 10, 64),
    (16, 128, 77, 5, 5, 64), (2, 1024, 77, 10, 10, 64), (1, 4096, 20, 5, 5, 64), (1, 500, 2000, 6, 2, 128), (1, 1000, 1, 4, 4, 64),
    (4, 17, 515, 24, 8, 64), (5, 2, 300, 7, 7, 64), (1, 100, 192, 9, 3, 64), (2, 640, 256, 2, 2, 128),
    (16, 2, 1500, 7, 7, 64), (3, 400, 1700, 8, 1, 64), (7, 77, 1600, 3, 3, 128), (74, 1, 600, 2, 1, 64), (1, 2000, 700, 8, 2, 128),
    (1, 3, 200, 64, 1, 64), (2, 5, 300, 128, 1, 128), (1, 9, 100, 256, 1, 64), (2, 1, 2100, 96, 1, 128), (1, 40, 130, 40, 1, 64)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("B,Sq,Skv,Hq,Hkv,D", CROSS)
def test_cross(ctx, layers, B, Sq, Skv, Hq, Hkv, D, dtype):
    g = gen(Sq * 7 + Skv)
    dt = DT[dtype]
    q, k, v = normal(g, B, Sq, Hq, D, dt=dt), normal(g, B, Skv, Hkv, D, dt=dt), normal(g, B, Skv, Hkv, D, dt=dt)
    check(layers.cross_attention(ctx, q, k, v), *cross_ref(q, k, v), "all keys")
    kv_len = torch.randint(0, Skv + 1, (B,), generator=g, device="cuda").int()
    mask = (torch.rand(B, Skv, generator=g, device="cuda") < 0.7)
    q_len = torch.randint(0, Sq + 1, (B,), generator=g, device="cuda").int()
    out = normal(g, B, Sq, Hq, D, dt=dt)
    ref = cross_ref(q, k, v, kv_len, q_len, mask, 0.2, out)
    check(layers.cross_attention(ctx, q, k, v, kv_len=kv_len, q_len=q_len, key_mask=mask, scale=0.2, out=out), *ref, "lengths, mask")
    assert ctx.fault() == 0


@pytest.mark.parametrize("Sq", [1, 200])
@pytest.mark.parametrize("Skv", [77, 1000])
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("D", [64, 128])
def test_cross_masked_places_may_hold_anything(ctx, layers, Sq, Skv, poison, D):
    g = gen(Sq + Skv)
    B, Hn = 4, 3
    q, k, v = (normal(g, B, n, Hn, D) for n in (Sq, Skv, Skv))
    kv_len = torch.tensor([Skv, Skv // 2, 1, 0], dtype=torch.int32, device="cuda")
    mask = torch.rand(B, Skv, generator=g, device="cuda") < 0.5
    mask[:, :70] = False  # the first whole tile of keys is masked
    mask[0, 71] = True
    ref = cross_ref(q, k, v, kv_len, None, mask)
    off = ~mask | (torch.arange(Skv, device="cuda") >= kv_len[:, None])
    k[off], v[off] = poison, poison
    check(layers.cross_attention(ctx, q, k, v, kv_len=kv_len, key_mask=mask), *ref)
    ref = cross_ref(q, torch.nan_to_num(k, 0, 0, 0), torch.nan_to_num(v, 0, 0, 0), kv_len * 0)
    assert (layers.cross_attention(ctx, q, k, v, kv_len=kv_len * 0) == 0).all()
    low = torch.full_like(k, -65504.0)  # the type's lowest value in a masked place
    k2, v2 = torch.where(off[..., None, None], low, k), torch.where(off[..., None, None], low, v)
    check(layers.cross_attention(ctx, q, k2, v2, kv_len=kv_len, key_mask=mask), *cross_ref(q, k2, v2, kv_len, None, mask))


@pytest.mark.parametrize("Sq", [1, 150])
def test_cross_lengths_outside_the_range_are_clamped(ctx, layers, Sq):
    g = gen(8)
    q, k, v = normal(g, 3, Sq, 2, 64), normal(g, 3, 90, 2, 64), normal(g, 3, 90, 2, 64)
    kv_len = torch.tensor([1000, -5, 90], dtype=torch.int32, device="cuda")
    q_len = torch.tensor([1000, Sq, -7], dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 3.0)
    ref = cross_ref(q, k, v, kv_len, q_len, None, None, out)
    check(layers.cross_attention(ctx, q, k, v, kv_len=kv_len, q_len=q_len, out=out), *ref)
    assert (out[2] == 3.0).all()


@pytest.mark.parametrize("Sq,Skv", [(1, 700), (300, 77), (150, 500)])
@pytest.mark.parametrize("D", [64, 128])
def test_cross_layouts(ctx, layers, Sq, Skv, D):
    """Head-major tensors, slices of fused projections, keys expanded over the batch, an output inside a larger one."""
    g = gen(9)
    B, Hq, Hkv = 3, 4, 2
    q = normal(g, B, Hq, Sq, D).transpose(1, 2)
    kv = normal(g, 1, Skv, 3, Hkv, D)
    k, v = kv[:, :, 0].expand(B, -1, -1, -1), kv[:, :, 2].expand(B, -1, -1, -1)
    hold = torch.full((B, Sq, Hq + 2, D), 9.0, dtype=torch.float16, device="cuda")
    out = hold[:, :, 1:-1]
    layers.cross_attention(ctx, q, k, v, out=out)
    check(out, *cross_ref(q, k, v))
    assert (hold[:, :, 0] == 9.0).all() and (hold[:, :, -1] == 9.0).all()
    k = k[:, :, :1].expand(-1, -1, Hkv, -1)  # one key head for all
    check(layers.cross_attention(ctx, q, k, v), *cross_ref(q, k, v))


@pytest.mark.parametrize("Sq,Skv", [(1, 3000), (5, 64), (200, 300), (130, 77)])
def test_cross_large_scores(ctx, layers, Sq, Skv):
    """Scores far apart (rising towards the end, so the running maximum moves often) and rows with one dominant key."""
    g = gen(11)
    q, k, v = normal(g, 2, Sq, 3, 64, scale=4.0), normal(g, 2, Skv, 3, 64), normal(g, 2, Skv, 3, 64)
    k = (k.float() * torch.linspace(0.1, 6.0, Skv, device="cuda")[None, :, None, None]).half()
    check(layers.cross_attention(ctx, q, k, v), *cross_ref(q, k, v))


@pytest.mark.parametrize("Sq,Skv", [(1, 3000), (3, 200), (300, 700), (260, 1290), (130, 128)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("order", ["rising", "falling", "saw"])
def test_cross_maximum_moves_in_every_tile(ctx, layers, Sq, Skv, D, order):
    """Scores that rise by some 12 per 128 keys: what was summed before is scaled down again and again."""
    g = gen(16)
    q, k, v = normal(g, 2, Sq, 2, D, scale=0.5), normal(g, 2, Skv, 2, D), normal(g, 2, Skv, 2, D)
    at = torch.arange(Skv, device="cuda").float()
    ramp = {"rising": at, "falling": Skv - at, "saw": at + (at % 128 < 40) * 300}[order] * 0.1
    q[..., 0] = 16.0
    k[..., 0] = (ramp * D ** 0.5 / 16)[None, :, None].half()
    check(layers.cross_attention(ctx, q, k, v), *cross_ref(q, k, v))
    lens = torch.tensor([Skv, max(1, Skv - 70)], dtype=torch.int32, device="cuda")
    mask = torch.rand(2, Skv, generator=g, device="cuda") < 0.5
    check(layers.cross_attention(ctx, q, k, v, kv_len=lens, key_mask=mask), *cross_ref(q, k, v, lens, None, mask))
    assert ctx.fault() == 0


@pytest.mark.parametrize("Sq,Skv", [(1, 3000), (40, 77), (300, 600)])
def test_cross_repeats_bit_for_bit(ctx, layers, Sq, Skv):
    g = gen(12)
    q, k, v = normal(g, 2, Sq, 8, 128), normal(g, 2, Skv, 4, 128), normal(g, 2, Skv, 4, 128)
    first = layers.cross_attention(ctx, q, k, v)
    for _ in range(3):
        assert torch.equal(layers.cross_attention(ctx, q, k, v), first)


@pytest.mark.parametrize("B,Sq,Skv,G,Hkv,D", [(3, 279, 371, 1, 2, 128), (4, 125, 328, 3, 1, 128), (2, 500, 700, 1, 3, 64), (6, 1, 900, 4, 2, 128),
                                              (6, 3, 900, 2, 2, 64), (8, 600, 77, 1, 5, 64)])
def test_cross_back_to_back(ctx, layers, B, Sq, Skv, G, Hkv, D):
    """Thirty calls queued at once, ragged lengths: every one gives the same bits, and the right ones."""
    g = gen(Sq)
    q, k, v = normal(g, B, Sq, G * Hkv, D), normal(g, B, Skv, Hkv, D), normal(g, B, Skv, Hkv, D)
    lens = torch.randint(0, Skv + 1, (B,), generator=g, device="cuda").int()
    outs = [layers.cross_attention(ctx, q, k, v, kv_len=lens) for _ in range(30)]
    check(outs[0], *cross_ref(q, k, v, lens))
    for o in outs[1:]:
        assert torch.equal(o, outs[0])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens", [[1500, 100] * 8, [100] * 15 + [1500], [1500, 1, 0, 128, 1500, 130, 64, 1500] * 2])
def test_cross_keys_of_one_tile_in_a_row(ctx, layers, lens, D):
    """Keys shared out over the card, some requests with a single tile for each of their heads: only one of a block's groups
    of warps has work, many times in a row."""
    g = gen(17)
    q, k, v = normal(g, 16, 2, 7, D), normal(g, 16, 1500, 7, D), normal(g, 16, 1500, 7, D)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    outs = [layers.cross_attention(ctx, q, k, v, kv_len=n) for _ in range(5)]
    for o in outs:
        check(o, *cross_ref(q, k, v, n))
    assert ctx.fault() == 0


@pytest.mark.parametrize("Sq", [1, 140])
def test_cross_offsets_past_32_bits(ctx, layers, Sq):
    """Keys and values whose offsets pass 2^32 elements (a token stride of 2^21 over 2100 tokens)."""
    g = gen(13)
    Skv, st = 2100, 1 << 21
    hold = torch.empty(Skv * st, dtype=torch.float16, device="cuda")
    kv = torch.as_strided(hold, (1, Skv, 2, 64), (Skv * st, st, 64, 1))
    kv.copy_(normal(g, 1, Skv, 2, 64))
    q = normal(g, 1, Sq, 1, 64)
    k, v = kv[:, :, :1], kv[:, :, 1:]
    check(layers.cross_attention(ctx, q, k, v), *cross_ref(q, k.contiguous(), v.contiguous()))


def test_cross_c_entry_refusals(ctx, dib):
    import ctypes
    L = dib.lib()
    q = torch.zeros(2, 3, 4, 64, dtype=torch.float16, device="cuda")
    ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")

    def call(**k):
        c = dict(B=2, H=4, Hkv=4, Sq=3, Skv=3, D=64)
        st = {n: (768, 256, 64) for n in ("qs", "ks", "vs", "os")}
        v = dict(dtype=1, cfg=None, scale=0.125, Q=q.data_ptr(), K=q.data_ptr(), V=q.data_ptr(), O=q.data_ptr(), ql=None, kl=None,
                 mask=None, ws=ws.data_ptr(), n=ws.numel())
        for key, val in k.items():
            (c if key in c else st if key in st else v)[key] = val
        v["cfg"] = (ctypes.c_longlong * 18)(*c.values(), *(s for t in st.values() for s in t))
        return L.di_cross_attention(ctx.h, *v.values())

    for bad in (dict(dtype=0), dict(B=0), dict(Sq=0), dict(Sq=-1), dict(Skv=0), dict(Skv=1 << 33), dict(H=0), dict(Hkv=3), dict(Q=None),
                dict(K=q.data_ptr() + 2), dict(ks=(768, 252, 64)), dict(qs=(-768, 256, 64)), dict(os=(0, 256, 64)),
                dict(os=(768, 0, 64)), dict(os=(768, 256, 0)), dict(ks=(768, 0, 64)), dict(scale=0.0), dict(scale=-1.0),
                dict(scale=float("nan")), dict(scale=float("inf"))):
        assert call(**bad) == dib.DI_EINVAL, bad
    assert call(D=96) == dib.DI_EUNSUPPORTED


# ---- together, streams, graphs --------------------------------------------------------------------------------

def layer_inputs(g, B, S, C, Skv, Cctx, dt):
    L, r, D = 4, 16, 64
    s = dict(x=normal(g, B * S, C, dt=dt), ctx=normal(g, B * Skv, Cctx, dt=dt))
    for n, (o, i) in dict(q=(C, C), kv=(2 * C, Cctx), o=(C, C)).items():
        s["w" + n], s["a" + n] = normal(g, o, i, dt=dt, scale=i ** -0.5), normal(g, L, r, i, dt=dt, scale=i ** -0.5)
        s["b" + n] = normal(g, L, o, r, dt=dt, scale=r ** -0.5)
    s["scale"] = torch.rand(L, generator=g, device="cuda")
    ids = torch.randint(-1, L, (B,), generator=g, device="cuda").int()
    s["rows"], s["ctx_rows"] = ids.repeat_interleave(S), ids.repeat_interleave(Skv)
    s["lens"] = torch.randint(1, Skv + 1, (B,), generator=g, device="cuda").int()
    s["gq"], s["gk"] = (1 + normal(g, D, dt=torch.float32, scale=0.2) for _ in range(2))
    side = int(S ** 0.5)
    at = torch.arange(S, device="cuda")
    s["pos"] = torch.stack([at // side, at % side], 1).int().contiguous()
    return s


def run_layer(ctx, layers, s, B, S, C, Skv):
    Hn = C // 64
    q = layers.linear_lora(ctx, s["x"], s["wq"], s["aq"], s["bq"], s["scale"], s["rows"]).view(B * S, Hn, 64)
    kv = layers.linear_lora(ctx, s["ctx"], s["wkv"], s["akv"], s["bkv"], s["scale"], s["ctx_rows"]).view(B * Skv, 2, Hn, 64)
    layers.qk_norm_rope(ctx, q, q_weight=s["gq"], positions=s["pos"], axis_dims=(32, 32), q_out=q)
    layers.qk_norm_rope(ctx, kv[:, 0], q_weight=s["gk"], q_out=kv[:, 0])
    kv = kv.view(B, Skv, 2, Hn, 64)
    o = layers.cross_attention(ctx, q.view(B, S, Hn, 64), kv[:, :, 0], kv[:, :, 1], kv_len=s["lens"])
    return layers.linear_lora(ctx, o.view(B * S, C), s["wo"], s["ao"], s["bo"], s["scale"], s["rows"], residual=s["x"])


def layer_ref(s, B, S, C, Skv):
    d = {k: v.double() if v.is_floating_point() else v for k, v in s.items()}
    Hn = C // 64

    def lin(x, n, rows, res=0):
        y = x @ d["w" + n].T + res
        for i in range(len(d["scale"])):
            y = y + (rows == i)[:, None] * d["scale"][i] * (x @ d["a" + n][i].T @ d["b" + n][i].T)
        return y

    def norm(x, w):
        return x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + 1e-6) * w

    q = norm(lin(d["x"], "q", s["rows"]).view(B * S, Hn, 64), d["gq"])
    fr = 10000.0 ** (-torch.arange(0, 32, 2, device="cuda").double() / 32)
    ang = torch.cat([s["pos"][:, a, None].double() * fr for a in range(2)], 1).repeat(B, 1)[:, None]
    q = torch.view_as_real(torch.view_as_complex(q.unflatten(-1, (32, 2)).contiguous()) * torch.polar(torch.ones_like(ang), ang)).flatten(-2)
    kv = lin(d["ctx"], "kv", s["ctx_rows"]).view(B, Skv, 2, Hn, 64)
    k, v = norm(kv[:, :, 0], d["gk"]), kv[:, :, 1]
    sc = torch.einsum("bihd,bjhd->bhij", q.view(B, S, Hn, 64), k) / 8
    sc = sc.masked_fill((torch.arange(Skv, device="cuda") >= s["lens"][:, None])[:, None, None], -math.inf)
    o = torch.einsum("bhij,bjhd->bihd", torch.softmax(sc, -1), v).reshape(B * S, C)
    return lin(o, "o", s["rows"], d["x"])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("B,S,C,Skv,Cctx", [(3, 64, 320, 77, 1024), (2, 1024, 640, 77, 1024), (5, 1, 320, 300, 64)])
def test_a_layer_of_them(ctx, layers, B, S, C, Skv, Cctx, dtype):
    """Projections, norms, attention and output projection in a row: the five 16-bit roundings on the way (h each, of
    values of order one that the softmax and two products pass on with a gain of about one) stay under 24 h of the result's
    size."""
    s = layer_inputs(gen(B * S), B, S, C, Skv, Cctx, DT[dtype])
    got, ref = run_layer(ctx, layers, s, B, S, C, Skv).double(), layer_ref(s, B, S, C, Skv)
    assert float((got - ref).abs().max()) <= 24 * H[DT[dtype]] * float(ref.abs().max())
    assert float((got - ref).norm() / ref.norm()) <= 2 * H[DT[dtype]]
    assert ctx.fault() == 0


@pytest.mark.parametrize("S", [1, 64])
def test_two_graphs_on_two_streams(dib, layers, S):
    """Two graphs captured from two contexts, replayed at once with new inputs, give what direct calls give: they share no
    scratch, and lengths, adapters and values are read at replay."""
    B, C, Skv, Cctx = 4, 320, 700, 320
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    ctxs = [dib.Context(0, stream=st) for st in streams]
    states, graphs, outs = [], [], []
    for i, (st, c) in enumerate(zip(streams, ctxs)):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            s = layer_inputs(gen(i), B, S, C, Skv, Cctx, torch.float16)
            run_layer(c, layers, s, B, S, C, Skv)
        st.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            o = run_layer(c, layers, s, B, S, C, Skv)
        states.append(s), graphs.append(g), outs.append(o)
    for r in range(3):
        new = [layer_inputs(gen(10 * r + i + 5), B, S, C, Skv, Cctx, torch.float16) for i in range(2)]
        for s, n in zip(states, new):
            for key in s:
                s[key].copy_(n[key])
        torch.cuda.synchronize()
        for _ in range(5):
            for st, g in zip(streams, graphs):
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        for s, o, c in zip(states, outs, ctxs):
            with torch.cuda.stream(c.stream):
                assert torch.equal(o, run_layer(c, layers, s, B, S, C, Skv))
            c.stream.synchronize()
    assert all(c.fault() == 0 for c in ctxs)


def test_results_belong_to_the_contexts_stream(dib, layers):
    """Called while another stream is current: the launches and the new tensors are the context's stream's."""
    st = torch.cuda.Stream()
    c = dib.Context(0, stream=st)
    s = lora_case(21, 40, 320, 320, 16, 3, torch.float16)
    ref = lora_ref(s)
    torch.cuda.synchronize()
    outs = [layers.linear_lora(c, **s) for _ in range(50)]
    st.synchronize()
    for o in outs:
        check(o, *ref)
    assert c.fault() == 0


def test_many_shapes_in_a_row(ctx, layers):
    """Fifty calls of changing shapes without a wait in between, each against its formula."""
    rng = np.random.default_rng(3)
    done = []
    for i in range(50):
        M, K, N, r, L = int(rng.integers(1, 400)), 64 * int(rng.integers(1, 12)), 16 * int(rng.integers(1, 40)), 8 * int(rng.integers(1, 17)), int(rng.integers(1, 20))
        s = lora_case(i, M, K, N, r, L, (torch.float16, torch.bfloat16)[i % 2], res=i % 3 == 0)
        done.append((layers.linear_lora(ctx, **s), *lora_ref(s)))
        B, Sq, Skv, G, Hkv, D = (int(v) for v in (rng.integers(1, 5), rng.integers(1, 300), rng.integers(1, 400), rng.integers(1, 4), rng.integers(1, 4), 64 * rng.integers(1, 3)))
        g = gen(i)
        q, k, v = normal(g, B, Sq, G * Hkv, D), normal(g, B, Skv, Hkv, D), normal(g, B, Skv, Hkv, D)
        lens = torch.randint(0, Skv + 1, (B,), generator=g, device="cuda").int()
        done.append((layers.cross_attention(ctx, q, k, v, kv_len=lens), *cross_ref(q, k, v, lens)))
    for got, ref, tol in done:
        check(got, ref, tol)
    assert ctx.fault() == 0
