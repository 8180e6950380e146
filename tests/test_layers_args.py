"""Refusals of the layers module: every bad argument raises DIError naming the operator before anything reaches the
device (the checks run on any machine: the tensors here are CPU tensors, which valid arguments end at)."""
from __future__ import annotations

import importlib
import types

import pytest
import torch


@pytest.fixture(scope="module")
def layers(dib):
    return importlib.import_module("draw_instant_b200.layers")


CTX = types.SimpleNamespace(device=0, h=None)


def lora_args(M=4, K=64, N=32, L=2, r=8, dt=torch.float16):
    return dict(x=torch.zeros(M, K, dtype=dt), w=torch.zeros(N, K, dtype=dt), a=torch.zeros(L, r, K, dtype=dt),
                b=torch.zeros(L, N, r, dtype=dt), scale=torch.zeros(L), row_adapter=torch.zeros(M, dtype=torch.int32))


def qk_args(T=4, H=2, D=64, dt=torch.float16):
    return dict(q=torch.zeros(T, H, D, dtype=dt), k=torch.zeros(T, H, D, dtype=dt), q_weight=torch.ones(D),
                k_weight=torch.ones(D), positions=torch.zeros(T, 2, dtype=torch.int32), axis_dims=(D // 2, D // 2))


def cross_args(B=2, Sq=3, Skv=5, H=4, Hkv=2, D=64, dt=torch.float16):
    return dict(q=torch.zeros(B, Sq, H, D, dtype=dt), k=torch.zeros(B, Skv, Hkv, D, dtype=dt),
                v=torch.zeros(B, Skv, Hkv, D, dtype=dt))


ARGS = {"linear_lora": lora_args, "qk_norm_rope": qk_args, "cross_attention": cross_args}

BAD = [
    ("linear_lora", dict(x=torch.zeros(4, 64)), "float16 or bfloat16"),
    ("linear_lora", dict(x=torch.zeros(4, 128, dtype=torch.float16)), "w must be"),
    ("linear_lora", dict(x=torch.zeros(0, 64, dtype=torch.float16)), "empty"),
    ("linear_lora", dict(x=torch.zeros(64, 4, dtype=torch.float16).T), "contiguous rows"),
    ("linear_lora", dict(w=torch.zeros(32, 64, dtype=torch.bfloat16)), "w must be"),
    ("linear_lora", dict(a=torch.zeros(2, 8, 32, dtype=torch.float16)), "a must be"),
    ("linear_lora", dict(b=torch.zeros(2, 8, 32, dtype=torch.float16)), "b must be"),
    ("linear_lora", dict(b=torch.zeros(2, 8, 32, dtype=torch.float16).transpose(1, 2)), "b must be"),
    ("linear_lora", dict(scale=torch.zeros(3)), "scale must be"),
    ("linear_lora", dict(scale=torch.zeros(2, dtype=torch.float64)), "scale must be"),
    ("linear_lora", dict(row_adapter=torch.zeros(4, dtype=torch.int64)), "row_adapter must be"),
    ("linear_lora", dict(row_adapter=torch.zeros(3, dtype=torch.int32)), "row_adapter must be"),
    ("linear_lora", dict(bias=torch.zeros(32, dtype=torch.float16)), "bias must be"),
    ("linear_lora", dict(residual=torch.zeros(4, 31, dtype=torch.float16)), "residual must be"),
    ("linear_lora", dict(out=torch.zeros(5, 32, dtype=torch.float16)), "out must be"),
    ("linear_lora", dict(act="relu"), "act must be"),
    ("qk_norm_rope", dict(q=torch.zeros(4, 2, 64)), "float16 or bfloat16"),
    ("qk_norm_rope", dict(q=torch.zeros(4, 128, dtype=torch.float16)), "axes"),
    ("qk_norm_rope", dict(q=torch.zeros(4, 2, 80, dtype=torch.float16)), "head dim"),
    ("qk_norm_rope", dict(q=torch.zeros(0, 2, 64, dtype=torch.float16)), "empty"),
    ("qk_norm_rope", dict(q=torch.zeros(2, 4, 64, dtype=torch.float16).transpose(0, 1)), "contiguous"),
    ("qk_norm_rope", dict(k=torch.zeros(5, 2, 64, dtype=torch.float16)), "tokens of q"),
    ("qk_norm_rope", dict(k=torch.zeros(4, 2, 64, dtype=torch.bfloat16)), "k must be"),
    ("qk_norm_rope", dict(k=None, k_out=torch.zeros(4, 2, 64, dtype=torch.float16)), "k_out without k"),
    ("qk_norm_rope", dict(q_weight=torch.ones(32)), "q_weight must be"),
    ("qk_norm_rope", dict(k_weight=torch.ones(64, dtype=torch.float16)), "k_weight must be"),
    ("qk_norm_rope", dict(axis_dims=(32, 16)), "axis_dims"),
    ("qk_norm_rope", dict(axis_dims=(33, 31)), "axis_dims"),
    ("qk_norm_rope", dict(axis_dims=(16, 16, 16, 16)), "axis_dims"),
    ("qk_norm_rope", dict(positions=None), "without positions"),
    ("qk_norm_rope", dict(positions=torch.zeros(4, 2)), "positions must be"),
    ("qk_norm_rope", dict(positions=torch.zeros(4, 3, dtype=torch.int32)), "positions must be"),
    ("qk_norm_rope", dict(positions=torch.zeros(0, 2, dtype=torch.int32)), "positions"),
    ("qk_norm_rope", dict(pairing="pairs"), "pairing"),
    ("qk_norm_rope", dict(theta=0.0), "theta"),
    ("qk_norm_rope", dict(q_out=torch.zeros(4, 3, 64, dtype=torch.float16)), "q_out"),
    ("cross_attention", dict(q=torch.zeros(2, 3, 4, 64)), "float16 or bfloat16"),
    ("cross_attention", dict(q=torch.zeros(3, 4, 64, dtype=torch.float16)), "axes"),
    ("cross_attention", dict(q=torch.zeros(2, 3, 3, 64, dtype=torch.float16)), "multiple"),
    ("cross_attention", dict(q=torch.zeros(2, 3, 4, 96, dtype=torch.float16)), "head dim"),
    ("cross_attention", dict(q=torch.zeros(2, 0, 4, 64, dtype=torch.float16)), "empty"),
    ("cross_attention", dict(k=torch.zeros(2, 5, 2, 128, dtype=torch.float16)), "alike"),
    ("cross_attention", dict(k=torch.zeros(1, 5, 2, 64, dtype=torch.float16)), "alike"),
    ("cross_attention", dict(v=torch.zeros(2, 6, 2, 64, dtype=torch.float16)), "alike"),
    ("cross_attention", dict(v=torch.zeros(2, 5, 2, 64, dtype=torch.bfloat16)), "v must be"),
    ("cross_attention", dict(v=torch.zeros(2, 5, 64, 2, dtype=torch.float16).transpose(2, 3)), "v must be"),
    ("cross_attention", dict(kv_len=torch.zeros(2, dtype=torch.int64)), "kv_len must be"),
    ("cross_attention", dict(kv_len=torch.zeros(3, dtype=torch.int32)), "kv_len must be"),
    ("cross_attention", dict(q_len=torch.zeros(2)), "q_len must be"),
    ("cross_attention", dict(key_mask=torch.zeros(2, 4, dtype=torch.uint8)), "key_mask must be"),
    ("cross_attention", dict(key_mask=torch.zeros(2, 5)), "key_mask must be"),
    ("cross_attention", dict(scale=0.0), "scale"),
    ("cross_attention", dict(scale=float("nan")), "scale"),
    ("cross_attention", dict(out=torch.zeros(2, 3, 2, 64, dtype=torch.float16)), "out must have"),
]


@pytest.mark.parametrize("op,change,says", BAD, ids=lambda v: v if isinstance(v, str) else "+".join(v) if isinstance(v, dict) else None)
def test_refuses(layers, dib, op, change, says):
    with pytest.raises(dib.DIError, match=says) as e:
        getattr(layers, op)(CTX, **{**ARGS[op](), **change})
    assert op in str(e.value)


@pytest.mark.parametrize("op", list(ARGS))
def test_valid_arguments_end_at_the_device(layers, dib, op):
    """No CPU path: arguments that pass every check are refused for their device."""
    with pytest.raises(dib.DIError, match="CUDA tensors"):
        getattr(layers, op)(CTX, **ARGS[op]())


def test_null_context_is_refused(dib):
    import ctypes
    L, cfg = dib.lib(), (ctypes.c_longlong * 18)(*([1] * 18))
    assert L.di_linear_lora(None, 1, cfg, *([None] * 10), 0) == dib.DI_EINVAL
    assert L.di_qk_norm_rope(None, 1, cfg, 0.0, 1.0, *([None] * 7)) == dib.DI_EINVAL
    assert L.di_cross_attention(None, 1, cfg, 1.0, *([None] * 8), 0) == dib.DI_EINVAL
    assert L.di_linear_lora_workspace(None, cfg) == 0 and L.di_cross_attention_workspace(None, cfg) == 0


def test_signatures_are_told_apart(layers):
    """The kept checks of one call are not another's: shapes, strides and types are all in the signature."""
    x = torch.zeros(4, 64, dtype=torch.float16)
    sigs = [layers._sig(t) for t in (x, x[:2], torch.zeros(4, 128, dtype=torch.float16)[:, :64], x.bfloat16(), x.T, None)]
    assert len(set(sigs)) == len(sigs)
