"""linear_lora, tiles whose rows name several adapters, with rows and adapters that are not finite: every row from its own
terms alone, and in a bounded time.  Formulas and tolerances are those of test_gpu_layers.py."""
from __future__ import annotations

import importlib

import pytest
import torch

from test_gpu_layers import DT, check, lora_case, lora_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def layers(dib):
    return importlib.import_module("draw_instant_b200.layers")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("M,per,K,N,r,L", [(129, 1, 64, 16, 8, 3), (300, 7, 320, 336, 24, 5), (257, 40, 192, 96, 72, 4), (700, 77, 640, 560, 128, 6),
                                           (1001, 33, 128, 2064, 40, 40)])
def test_rows_beside_those_that_are_not_finite(ctx, layers, M, per, K, N, r, L, dtype):
    """One request of NaN, an infinity in another's row and two adapters that hold them: only the rows that they reach show
    it, and the others, computed again, are right with bias, activation and residual."""
    rows = [(m // per * 5) % (L + 1) - 1 for m in range(M)]
    s = lora_case(M + r, M, K, N, r, L, DT[dtype], res=True, rows=rows)
    names = s["row_adapter"]
    ref, tol = lora_ref(s, "gelu")
    gone = torch.zeros(M, dtype=torch.bool, device="cuda")
    s["x"][per:2 * per], gone[per:2 * per] = float("nan"), True
    s["x"][M - 1, K - 1], gone[M - 1] = float("inf"), True
    s["b"][1], s["a"][2] = float("inf"), float("nan")
    gone |= (names == 1) | (names == 2)
    assert gone.any() and not gone.all()
    got = layers.linear_lora(ctx, **s, act="gelu")
    check(got[~gone], ref[~gone], tol[~gone])
    assert torch.isnan(got[per:2 * per]).all() and torch.isnan(got[names == 2]).all()
    assert not torch.isfinite(got[names == 1]).any()
    assert ctx.fault() == 0


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("M,r", [(60, 16), (300, 16), (300, 104)])
def test_an_infinity_in_an_adapter_stays_one(ctx, layers, M, r, dtype):
    """One infinite value of B: the column of the rows that name the adapter is infinite, with the sign of the inner value."""
    s = lora_case(r, M, 320, 48, r, 3, DT[dtype], rows=[m // 7 % 3 for m in range(M)])
    s["b"][1, 5, 3] = float("inf")
    mine = s["row_adapter"] == 1
    t = s["x"].double() @ s["a"][1, 3].double()
    clear = mine & (t.abs() > 1e-2)
    assert clear.sum() > 10
    got = layers.linear_lora(ctx, **s)
    assert torch.equal(got[clear, 5].double(), t[clear].sign() * float("inf"))
    s["b"][1, 5, 3] = 0
    ref, tol = lora_ref(s)
    other = torch.arange(48, device="cuda") != 5
    check(got[:, other], ref[:, other], tol[:, other])
    check(got[~mine], ref[~mine], tol[~mine])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("M,K,N,r,L", [(256, 320, 336, 16, 256), (300, 128, 64, 128, 300), (513, 64, 32, 8, 400), (192, 640, 2048, 64, 192)])
def test_every_row_with_an_adapter_of_its_own(ctx, layers, M, K, N, r, L, dtype):
    """More adapters in a tile than its lists hold entries for, three of 32 adapters or of 256 / rank: the lists are used again
    and again within one tile."""
    s = lora_case(M, M, K, N, r, L, DT[dtype], res=M % 2 == 0, rows=[(m * 7 + 3) % L for m in range(M)])
    first = layers.linear_lora(ctx, **s)
    check(first, *lora_ref(s))
    for _ in range(3):
        assert torch.equal(layers.linear_lora(ctx, **s), first)
    assert ctx.fault() == 0


@pytest.mark.parametrize("M,per,K,N,r,L", [(1001, 77, 1024, 4096, 64, 6), (512, 77, 4096, 4096, 128, 8)])
def test_rows_that_are_not_finite_do_not_hold_up_the_batch(ctx, layers, M, per, K, N, r, L):
    """With every row affected, each warp takes its three chunks again in four parts of 16 rows and columns: K / 32 steps of
    some 600 cycles and a step or two for every adapter, 0.04 to 0.16 ms a chunk for K of 1024 to 4096.  That is four to ten
    times the batch's 30 to 60 us, and never thirty times."""
    s = lora_case(1, M, K, N, r, L, torch.bfloat16, rows=[m // per % L for m in range(M)])
    out = torch.empty(M, N, dtype=torch.bfloat16, device="cuda")

    def time():
        best = 1e9
        for _ in range(5):
            a, b = torch.cuda.Event(True), torch.cuda.Event(True)
            a.record(ctx.stream)
            layers.linear_lora(ctx, **s, out=out)
            b.record(ctx.stream)
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    torch.cuda.synchronize()
    clean = time()
    s["x"].fill_(float("nan"))
    torch.cuda.synchronize()
    bad = time()
    assert torch.isnan(out).all()
    assert bad < 30 * max(clean, 0.03), f"{bad:.3f} ms, {clean:.3f} without"
