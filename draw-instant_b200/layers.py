"""Attention-layer operators for batches whose requests differ from one another, beside di_linear and di_attention:

linear_lora      a linear layer with a low-rank adapter per row beside the shared weight (di_linear_lora)
qk_norm_rope     RMS norm of query and key heads with the rotation by position axes (di_qk_norm_rope)
cross_attention  attention over an encoder's states with lengths and a key mask per request (di_cross_attention)

They take and return torch tensors on the context's device (fp16 or bf16 activations and weights, fp32 norm
weights, biases and scales, int32 indices) and launch on the context's stream without synchronising.  Scratch
memory is allocated by torch on that stream for each call, so calls on several streams, and graphs captured from
them, share none.  A result is the `out` that was passed, or a new tensor.  Bad arguments raise DIError.

    q = linear_lora(ctx, x, w_q, a_q, b_q, scale, rows).view(B * S, H, 64)
    qk_norm_rope(ctx, q, q_weight=g, positions=pos, axis_dims=(32, 32), q_out=q)
    o = cross_attention(ctx, q.view(B, S, H, 64), k, v, kv_len=prompt_lengths)

A call's checks and its cfg block depend on shapes, strides, types and devices alone.  They are kept per such
signature, so a repeated call costs one dictionary lookup before it launches.
"""
from __future__ import annotations

import ctypes

import torch

from . import DI_BF16, DI_F16, Context, DIError, lib

__all__ = ["linear_lora", "qk_norm_rope", "cross_attention"]

_CODE = {torch.float16: DI_F16, torch.bfloat16: DI_BF16}
_ACT = {"none": 0, "silu": 1, "gelu": 2}
_PAIRING = {"interleaved": 0, "halves": 1}
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)

# signature of a call -> (dtype code, cfg block, scratch bytes, shape of a new result, dtype)
_plans: dict = {}


def _keep(key, plan):
    if len(_plans) >= 4096:
        _plans.clear()
    _plans[key] = plan
    return plan


def _cfg(*vals):
    return (ctypes.c_longlong * len(vals))(*vals)


def _code(t, what: str) -> int:
    code = _CODE.get(t.dtype)
    if code is None:
        raise DIError(f"{what}: tensors must be float16 or bfloat16, got {t.dtype}")
    return code


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise DIError(what)


def _on(ctx: Context, what: str, *tensors) -> None:
    """Every tensor must live on the context's device (there is no CPU path)."""
    for t in tensors:
        if t is not None and t.get_device() != ctx.device:
            raise DIError(f"{what}: tensors must be CUDA tensors on device {ctx.device}, got one on {t.device}")


def _like(t, dtype, shape, what: str) -> None:
    """A contiguous tensor of this type and shape, or None."""
    if t is not None and (t.dtype != dtype or t.shape != shape or not t.is_contiguous()):
        raise DIError(f"{what} must be a contiguous {dtype} tensor of shape {tuple(shape)}, got {t.dtype} {tuple(t.shape)}")


def _new(ctx: Context, shape, dtype):
    """A tensor whose memory belongs to the context's stream."""
    st = ctx.stream
    now = _raw_stream(ctx.device) if _raw_stream else torch.cuda.current_stream(ctx.device).cuda_stream
    if now == st.cuda_stream:
        return torch.empty(shape, dtype=dtype, device=st.device)
    with torch.cuda.stream(st):
        return torch.empty(shape, dtype=dtype, device=st.device)


def _sig(t):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.get_device())


def _rows(t, shape, dtype, what: str):
    """A [.., n] tensor of contiguous rows; returns its row stride."""
    if t.dtype != dtype or t.shape != shape or (t.stride(1) != 1 and shape[1] > 1):
        raise DIError(f"{what} must be a {dtype} tensor of shape {tuple(shape)} with contiguous rows, "
                      f"got {t.dtype} {tuple(t.shape)} with strides {t.stride()}")
    return t.stride(0) if shape[0] > 1 else shape[1]


def linear_lora(ctx: Context, x, w, a, b, scale, row_adapter, bias=None, residual=None, act: str = "none", out=None):
    """act(x w^T + bias + scale[i] (x a[i]^T) b[i]^T) + residual with i = row_adapter[row], per row of x.

    x [M, K], w [N, K], a [L, r, K], b [L, N, r] (fp16 or bf16), scale [L] fp32, row_adapter [M] int32 on the
    device (negative: no adapter), bias [N] fp32, residual and out [M, N].  K a multiple of 64, N of 16, r of 8 up
    to 128: adapters of other ranks are padded with zeros.  x, residual and out may have a row stride; out may be
    the residual; it shares no other memory with x, the weights or a residual.  Rows may take the adapters in any order; from some hundred rows on, equal neighbours are fastest.
    act: none, silu or gelu, before the residual.  An index past the last adapter sets flag 16 in the context's fault
    word and counts as none.  In fp16, scale * (x a^T) has to stay inside the type's range."""
    key = (ctx.device, act, _sig(x), _sig(w), _sig(a), _sig(b), _sig(scale), _sig(row_adapter), _sig(bias), _sig(residual), _sig(out))
    plan = _plans.get(key)
    if plan is None:
        plan = _keep(key, _plan_lora(ctx, x, w, a, b, scale, row_adapter, bias, residual, act, out))
    code, cfg, n, shape, dt = plan
    if out is None:
        out = _new(ctx, shape, dt)
    ws = _new(ctx, n, torch.uint8) if n else None
    rc = lib().di_linear_lora(ctx.h, code, cfg, x.data_ptr(), w.data_ptr(), a.data_ptr(), b.data_ptr(), scale.data_ptr(),
                              row_adapter.data_ptr(), None if bias is None else bias.data_ptr(),
                              None if residual is None else residual.data_ptr(), out.data_ptr(),
                              None if ws is None else ws.data_ptr(), n)
    if rc:
        ctx.check(rc, "linear_lora")
    return out


def _plan_lora(ctx, x, w, a, b, scale, row_adapter, bias, residual, act, out):
    what = "linear_lora"
    code, dt = _code(x, what), x.dtype
    _need(x.dim() == 2 and w.dim() == 2 and a.dim() == 3 and b.dim() == 3, f"{what}: x and w are matrices, a and b have three axes")
    M, K = x.shape
    N, (L, r) = w.shape[0], a.shape[:2]
    _need(M > 0 and N > 0 and K > 0 and L > 0, f"{what}: empty tensors")
    _need(act in _ACT, f"{what}: act must be one of {', '.join(_ACT)}")
    ldx = _rows(x, (M, K), dt, f"{what}: x")
    _like(w, dt, (N, K), f"{what}: w")
    _like(a, dt, (L, r, K), f"{what}: a")
    _like(b, dt, (L, N, r), f"{what}: b")
    _like(scale, torch.float32, (L,), f"{what}: scale")
    _like(row_adapter, torch.int32, (M,), f"{what}: row_adapter")
    _like(bias, torch.float32, (N,), f"{what}: bias")
    ldr = 0 if residual is None else _rows(residual, (M, N), dt, f"{what}: residual")
    ldy = N if out is None else _rows(out, (M, N), dt, f"{what}: out")
    _on(ctx, what, x, w, a, b, scale, row_adapter, bias, residual, out)
    cfg = _cfg(M, N, K, r, L, ldx, ldr, ldy, _ACT[act])
    return code, cfg, lib().di_linear_lora_workspace(ctx.h, cfg), (M, N), dt


def _heads(t, dt, D, what: str):
    """A [T, H, D] tensor whose heads are contiguous; returns (H, token stride)."""
    _need(t.dim() == 3, f"{what} must have the axes [tokens, heads, head dim]")
    T, H, d = t.shape
    if t.dtype != dt or d != D or t.stride(2) != 1 or (H > 1 and t.stride(1) != D):
        raise DIError(f"{what} must be a {dt} tensor [tokens, heads, {D}] whose heads are contiguous, "
                      f"got {t.dtype} {tuple(t.shape)} with strides {t.stride()}")
    return H, (t.stride(0) if T > 1 else H * D)


def qk_norm_rope(ctx: Context, q, k=None, q_weight=None, k_weight=None, eps: float = 1e-6, positions=None, axis_dims=(),
                 theta: float = 10000.0, pairing: str = "interleaved", q_out=None, k_out=None):
    """Per head: x * rsqrt(mean(x^2) + eps) * weight, then the rotation by the token's positions; returns
    (q_out, k_out), or q_out alone when there is no k.

    q [T, Hq, D] and k [T, Hk, D] with D 64 or 128 (fp16 or bf16; tokens may be strided, as in a fused
    projection; q_out may be q and k_out may be k, and they share no other memory with them or each other).  q_weight, k_weight [D] fp32, None: no norm.  positions [P, n] int32
    on the device, token t takes row t % P, None: no rotation.  axis_dims: n = 1 to 3 even dims that sum to D, in
    the positions' order; pair j of axis a turns by positions[., a] * theta^(-2 j / axis_dims[a]).  pairing:
    "interleaved" (values 2i, 2i + 1) or "halves" (values i, i + D / 2)."""
    if not theta > 0:
        raise DIError("qk_norm_rope: theta must be positive")
    key = (ctx.device, pairing, tuple(axis_dims), _sig(q), _sig(k), _sig(q_weight), _sig(k_weight), _sig(positions), _sig(q_out), _sig(k_out))
    plan = _plans.get(key)
    if plan is None:
        plan = _keep(key, _plan_qk(ctx, q, k, q_weight, k_weight, positions, axis_dims, pairing, q_out, k_out))
    code, cfg = plan
    if q_out is None:
        q_out = _new(ctx, q.shape, q.dtype)
    if k is not None and k_out is None:
        k_out = _new(ctx, k.shape, q.dtype)
    rc = lib().di_qk_norm_rope(ctx.h, code, cfg, eps, theta, q.data_ptr(), None if k is None else k.data_ptr(),
                               None if q_weight is None else q_weight.data_ptr(),
                               None if k_weight is None else k_weight.data_ptr(),
                               None if positions is None else positions.data_ptr(), q_out.data_ptr(),
                               None if k is None else k_out.data_ptr())
    if rc:
        ctx.check(rc, "qk_norm_rope")
    return q_out if k is None else (q_out, k_out)


def _plan_qk(ctx, q, k, q_weight, k_weight, positions, axis_dims, pairing, q_out, k_out):
    what = "qk_norm_rope"
    code, dt = _code(q, what), q.dtype
    _need(q.dim() == 3, f"{what}: q must have the axes [tokens, heads, head dim]")
    T, _, D = q.shape
    _need(T > 0 and q.shape[1] > 0, f"{what}: empty tensors")
    _need(D in (64, 128), f"{what}: head dim must be 64 or 128, got {D}")
    _need(pairing in _PAIRING, f"{what}: pairing must be one of {', '.join(_PAIRING)}")
    Hq, ldq = _heads(q, dt, D, f"{what}: q")
    Hk = ldk = ldko = 0
    if k is not None:
        Hk, ldk = _heads(k, dt, D, f"{what}: k")
        _need(Hk > 0 and k.shape[0] == T, f"{what}: k must have the tokens of q and at least one head")
    else:
        _need(k_out is None, f"{what}: k_out without k")
    _like(q_weight, torch.float32, (D,), f"{what}: q_weight")
    _like(k_weight, torch.float32, (D,), f"{what}: k_weight")
    dims = tuple(axis_dims)
    P = 0
    if positions is not None:
        _need(1 <= len(dims) <= 3 and all(d > 0 and d % 2 == 0 for d in dims) and sum(dims) == D,
              f"{what}: axis_dims must be 1 to 3 even dims that sum to the head dim")
        _need(positions.dim() == 2 and positions.shape[0] > 0, f"{what}: positions must have the axes [rows, position axes]")
        P = positions.shape[0]
        _like(positions, torch.int32, (P, len(dims)), f"{what}: positions")
    else:
        _need(not dims, f"{what}: axis_dims without positions")
    ldqo = Hq * D
    if q_out is not None:
        _need(q_out.shape == q.shape, f"{what}: q_out must have the shape of q")
        ldqo = _heads(q_out, dt, D, f"{what}: q_out")[1]
    if k_out is not None:
        _need(k_out.shape == k.shape, f"{what}: k_out must have the shape of k")
        ldko = _heads(k_out, dt, D, f"{what}: k_out")[1]
    elif Hk:
        ldko = Hk * D
    _on(ctx, what, q, k, q_weight, k_weight, positions, q_out, k_out)
    return code, _cfg(T, Hq, Hk, D, ldq, ldk, ldqo, ldko, P, _PAIRING[pairing], len(dims), *(dims + (0, 0, 0))[:3])


def _bshd(t, dt, what: str):
    """Batch, token and head strides of a [B, S, H, D] tensor whose last axis is contiguous."""
    if t.dtype != dt or t.stride(3) != 1:
        raise DIError(f"{what} must be a {dt} tensor [batch, tokens, heads, head dim] with a contiguous last axis, "
                      f"got {t.dtype} {tuple(t.shape)} with strides {t.stride()}")
    return t.stride()[:3]


def cross_attention(ctx: Context, q, k, v, kv_len=None, q_len=None, key_mask=None, scale: float | None = None, out=None):
    """softmax(scale q k^T) v over each request's valid keys.

    q [B, Sq, H, D], k and v [B, Skv, Hkv, D] (fp16 or bf16), H a multiple of Hkv (query head h reads key head
    h / (H / Hkv)), D 64 or 128; any strides that are multiples of 8 elements with a contiguous last axis, so token-major
    and head-major layouts, slices of fused projections and keys and values expanded over the batch all go in place.
    Key j of request b is valid when j < kv_len[b] and key_mask[b, j] != 0 (kv_len [B] int32, key_mask [B, Skv] uint8 or
    bool, both on the device, None: all); what masked keys and values hold, infinities and NaN included, has no effect.
    A request without a valid key gives zeros.  Query rows from q_len[b] on (int32) are not computed:
    their rows of out stay as they were, and are zero in a new tensor.  The
    probabilities are rounded to the tensors' type for the product with v, all else is held in 32 bits: for ordinary values
    the result is off by up to 1.4 times its own rounding.  out may be q itself; it shares no other memory with q, k or v.
    scale: positive, 1 / sqrt(D) by default."""
    if scale is not None and not 0 < scale < float("inf"):
        raise DIError("cross_attention: scale must be positive and finite")
    key = (ctx.device, _sig(q), _sig(k), _sig(v), _sig(kv_len), _sig(q_len), _sig(key_mask), _sig(out))
    plan = _plans.get(key)
    if plan is None:
        plan = _keep(key, _plan_cross(ctx, q, k, v, kv_len, q_len, key_mask, out))
    code, cfg, n, default, _ = plan
    if scale is None:
        scale = default
    if out is None:
        out = _new(ctx, q.shape, q.dtype)
        if q_len is not None:  # rows that are not computed hold nothing of another tensor's
            with torch.cuda.stream(ctx.stream):
                out.zero_()
    ws = _new(ctx, n, torch.uint8) if n else None
    rc = lib().di_cross_attention(ctx.h, code, cfg, scale, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                                  None if q_len is None else q_len.data_ptr(), None if kv_len is None else kv_len.data_ptr(),
                                  None if key_mask is None else key_mask.data_ptr(), None if ws is None else ws.data_ptr(), n)
    if rc:
        ctx.check(rc, "cross_attention")
    return out


def _plan_cross(ctx, q, k, v, kv_len, q_len, key_mask, out):
    what = "cross_attention"
    code, dt = _code(q, what), q.dtype
    _need(q.dim() == 4 and k.dim() == 4 and v.dim() == 4, f"{what}: q, k and v must have the axes [batch, tokens, heads, head dim]")
    B, Sq, H, D = q.shape
    Skv, Hkv = k.shape[1:3]
    _need(B > 0 and Sq > 0 and H > 0 and Skv > 0 and Hkv > 0, f"{what}: empty tensors")
    _need(D in (64, 128), f"{what}: head dim must be 64 or 128, got {D}")
    _need(k.shape == (B, Skv, Hkv, D) and v.shape == k.shape, f"{what}: k and v must be [{B}, tokens, heads, {D}], alike")
    _need(H % Hkv == 0, f"{what}: the query heads must be a multiple of the key heads")
    strides = [_bshd(t, dt, f"{what}: {n}") for t, n in ((q, "q"), (k, "k"), (v, "v"))]
    _like(kv_len, torch.int32, (B,), f"{what}: kv_len")
    _like(q_len, torch.int32, (B,), f"{what}: q_len")
    if key_mask is not None and key_mask.dtype == torch.bool:
        key_mask = key_mask.view(torch.uint8)
    _like(key_mask, torch.uint8, (B, Skv), f"{what}: key_mask")
    if out is not None:
        _need(out.shape == q.shape, f"{what}: out must have the shape of q")
        strides.append(_bshd(out, dt, f"{what}: out"))
    else:
        strides.append((Sq * H * D, H * D, D))
    _on(ctx, what, q, k, v, kv_len, q_len, key_mask, out)
    cfg = _cfg(B, H, Hkv, Sq, Skv, D, *(s for t in strides for s in t))
    return code, cfg, lib().di_cross_attention_workspace(ctx.h, cfg), D ** -0.5, dt
