"""cross_attention with query lengths and no output tensor of the caller's: the rows that are not computed are zero."""
from __future__ import annotations

import importlib

import pytest
import torch

from test_gpu_layers import check, cross_ref, gen, normal

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def layers(dib):
    return importlib.import_module("draw_instant_b200.layers")


def soil(stream, like):
    """Leaves memory of this size full of NaN for the next tensor that the stream gets."""
    with torch.cuda.stream(stream):
        old = [torch.full_like(like, float("nan")) for _ in range(4)]
        del old


@pytest.mark.parametrize("B,Sq,Skv,H,Hkv,D", [(3, 200, 77, 5, 5, 64), (4, 1, 900, 8, 2, 128), (3, 130, 300, 4, 4, 128), (2, 7, 5, 2, 1, 64)])
def test_rows_behind_the_last_query_of_a_new_tensor_are_zero(ctx, layers, B, Sq, Skv, H, Hkv, D):
    g = gen(Sq)
    q, k, v = normal(g, B, Sq, H, D), normal(g, B, Skv, Hkv, D), normal(g, B, Skv, Hkv, D)
    q_len = torch.tensor([(Sq * i) // B for i in range(B)], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    soil(ctx.stream, q)
    got = layers.cross_attention(ctx, q, k, v, q_len=q_len)
    torch.cuda.synchronize()
    for b, n in enumerate(q_len.tolist()):
        assert (got[b, n:] == 0).all()
    check(got, *cross_ref(q, k, v, None, q_len))
    assert ctx.fault() == 0


def test_also_on_a_stream_of_its_own_and_in_a_graph(dib, layers):
    """Called while another stream is current, and replayed after its output was overwritten."""
    st = torch.cuda.Stream()
    c = dib.Context(0, stream=st)
    g = gen(5)
    q, k, v = normal(g, 3, 40, 2, 64), normal(g, 3, 90, 2, 64), normal(g, 3, 90, 2, 64)
    q_len = torch.tensor([40, 0, 13], dtype=torch.int32, device="cuda")
    ref = cross_ref(q, k, v, None, q_len)
    torch.cuda.synchronize()
    soil(st, q)
    got = layers.cross_attention(c, q, k, v, q_len=q_len)
    st.synchronize()
    check(got, *ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        got = layers.cross_attention(c, q, k, v, q_len=q_len)
    with torch.cuda.stream(st):
        got.fill_(float("nan"))
        graph.replay()
    st.synchronize()
    check(got, *ref)
    assert c.fault() == 0
