"""Outputs that share memory with inputs: what a call may do in place, and what it refuses (the checks are the host's: nothing
is launched)."""
from __future__ import annotations

import importlib

import pytest
import torch

from test_gpu_layers import check, cross_ref, gen, lora_case, lora_ref, normal, qk_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def layers(dib):
    return importlib.import_module("draw_instant_b200.layers")


@pytest.mark.parametrize("M", [1, 12, 300])
def test_lora_refuses_an_output_over_its_input(ctx, dib, layers, M):
    s = lora_case(M, M, 320, 320, 16, 3, torch.float16)
    wide = torch.zeros(M + 2, 960, dtype=torch.float16, device="cuda")
    x = wide[:M, :320]
    x.copy_(s["x"])
    s["x"] = x
    ref = lora_ref(s)
    bad = [x, wide[:M, 312:632], wide.view(-1)[8:8 + M * 320].view(M, 320)]
    bad += [wide[1:M + 1, :320], wide.view(-1)[960 - 312:960 - 312 + 960 * M].view(M, 960)[:, :320]] if M > 1 else []
    for out in bad:
        with pytest.raises(dib.DIError, match="shares memory"):
            layers.linear_lora(ctx, **s, out=out)
    for out in (wide[:M, 320:640], wide[:M, 640:], wide[1:M + 1, 320:640]):  # beside it, or behind the row before
        check(layers.linear_lora(ctx, **s, out=out), *ref)
    assert ctx.fault() == 0


@pytest.mark.parametrize("M", [1, 12, 300])
def test_lora_refuses_a_residual_that_is_partly_the_output(ctx, dib, layers, M):
    s = lora_case(M + 1, M, 320, 320, 16, 3, torch.bfloat16, res=True)
    ref = lora_ref(s)
    hold = torch.zeros(M + 1, 640, dtype=torch.bfloat16, device="cuda")
    y = hold[:M, :320]
    for other in ([hold[:M, 8:328]] + ([hold[1:, :320]] if M > 1 else [])):
        with pytest.raises(dib.DIError, match="shares memory"):
            layers.linear_lora(ctx, **{**s, "residual": other}, out=y)
    for other in (y, hold[:M, 320:]):
        other.copy_(s["residual"])
        check(layers.linear_lora(ctx, **{**s, "residual": other}, out=y), *ref)
    assert ctx.fault() == 0


@pytest.mark.parametrize("T", [1, 50, 3000])
@pytest.mark.parametrize("D", [64, 128])
def test_qk_refuses_outputs_over_other_heads(ctx, dib, layers, T, D):
    g = gen(T)
    x = normal(g, T + 1, 9, D)
    w = torch.ones(D, device="cuda")
    before = x.clone()
    q, k = x[:T, :3], x[:T, 3:5]
    bad = [dict(q_out=x[:T, 1:4]), dict(q_out=x[:T, 2:5]), dict(k_out=x[:T, 2:4]), dict(k_out=x[:T, 4:6]), dict(q_out=q, k_out=x[:T, 1:3]),
           dict(q_out=x[:T, 5:8], k_out=x[:T, 7:9])]
    bad += [dict(q_out=x[1:, :3]), dict(k_out=x[1:, 4:6])] if T > 1 else []
    for outs in bad:
        with pytest.raises(dib.DIError, match="shares memory"):
            layers.qk_norm_rope(ctx, q, k, q_weight=w, k_weight=w, **outs)
    torch.cuda.synchronize()
    assert torch.equal(x, before)
    y, z = layers.qk_norm_rope(ctx, q, k, q_weight=w, k_weight=w, q_out=q, k_out=x[:T, 5:7])  # in place, and beside
    check(y, *qk_ref(before[:T, :3], w, 1e-6, None, (), 1.0, "interleaved"))
    check(z, *qk_ref(before[:T, 3:5], w, 1e-6, None, (), 1.0, "interleaved"))
    assert torch.equal(x[:T, 3:5], before[:T, 3:5]) and torch.equal(x[:, 7:], before[:, 7:]) and torch.equal(x[T], before[T])
    assert ctx.fault() == 0


@pytest.mark.parametrize("B,Sq,Skv,H,Hkv,D", [(3, 500, 77, 5, 5, 64), (2, 700, 400, 4, 2, 128), (16, 1, 1500, 8, 2, 128), (7, 130, 1600, 3, 3, 64)])
def test_cross_in_place_of_the_queries(ctx, layers, B, Sq, Skv, H, Hkv, D):
    """Many queries, ragged ones, and keys shared out over the card: the queries lie in a wider buffer and become the result."""
    g = gen(Sq)
    hold = normal(g, B, Sq, H + 2, D)
    before = hold.clone()
    q, k, v = hold[:, :, 1:-1], normal(g, B, Skv, Hkv, D), normal(g, B, Skv, Hkv, D)
    q_len = torch.tensor([max(1, Sq - 3 * i) for i in range(B)], dtype=torch.int32, device="cuda")
    ref = cross_ref(q.contiguous(), k, v, None, q_len, None, None, q.contiguous())
    layers.cross_attention(ctx, q, k, v, q_len=q_len, out=q)
    check(q, *ref)
    assert torch.equal(hold[:, :, 0], before[:, :, 0]) and torch.equal(hold[:, :, -1], before[:, :, -1])
    assert ctx.fault() == 0


@pytest.mark.parametrize("Sq", [1, 40])
def test_cross_refuses_an_output_over_keys_and_values(ctx, dib, layers, Sq):
    g = gen(Sq)
    q, kv = normal(g, 3, Sq, 4, 64), normal(g, 3, Sq, 2, 4, 64)
    for out in (kv[:, :, 0], kv[:, :, 1]):
        with pytest.raises(dib.DIError, match="shares memory"):
            layers.cross_attention(ctx, q, kv[:, :, 0], kv[:, :, 1], out=out)
    other = q.view(3, 4, Sq, 64).transpose(1, 2)  # the queries' memory in another order
    if Sq > 1:
        with pytest.raises(dib.DIError, match="shares memory"):
            layers.cross_attention(ctx, q, kv[:, :, 0], kv[:, :, 1], out=other)
