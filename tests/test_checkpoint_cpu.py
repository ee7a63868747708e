"""Refusals of the checkpoint and attention entry points that need no GPU: everything is checked on the host before
anything is launched, so the made-up pointers are never followed."""
import ctypes

import pytest
import torch


def test_python_refusals():
    from tango_amd.checkpoint import pack
    from tango_amd.graph_attention import graph_attention
    with pytest.raises(RuntimeError, match="GPU"):
        pack(torch.zeros(4, 8))
    with pytest.raises(TypeError):
        pack([1.0])
    with pytest.raises(RuntimeError, match="GPU"):
        graph_attention(None, *(torch.zeros(2, 1, 4) for _ in range(3)))


def test_checkpoints_on_the_host_are_refused():
    from tango_amd.checkpoint import Packed, need_packed, unpack
    p = Packed(torch.zeros(4, 16, dtype=torch.int8), torch.zeros(4, 2), 8, (4, 16), torch.float32)
    with pytest.raises(RuntimeError, match="GPU"):
        unpack(p)
    with pytest.raises(TypeError):
        need_packed(p.values, "unpack")


@pytest.mark.parametrize("change", [
    dict(values=torch.zeros(4, 24)), dict(scale=torch.zeros(4, 3).double()), dict(scale=torch.zeros(4, 2)),
    dict(scale=torch.zeros(3, 4).t()), dict(values=torch.zeros(3, 24, dtype=torch.int8)), dict(values=torch.zeros(24, 4, dtype=torch.int8).t()),
    dict(values=torch.zeros(4, 16, dtype=torch.int8)), dict(group=0), dict(group=16), dict(group=8.0), dict(shape=(5, 24)),
    dict(shape=(4, 23)), dict(dtype=torch.float64),
])
def test_checkpoints_of_parts_that_do_not_fit(change):
    """A checkpoint put together by hand is checked, and its parts stay."""
    from tango_amd.checkpoint import Packed
    parts = dict(values=torch.zeros(4, 24, dtype=torch.int8), scale=torch.zeros(4, 3), group=8, shape=(2, 2, 24), dtype=torch.bfloat16)
    p = Packed(**parts)
    with pytest.raises(RuntimeError):
        Packed(**{**parts, **change})
    (name, value), = change.items()
    with pytest.raises(AttributeError):
        setattr(p, name, value)
    assert getattr(p, name) is parts[name]


def test_preparing_a_graph_that_was_not_preprocessed():
    from tango_amd.graph import Graph
    from tango_amd.graph_attention import prepare_attention
    with pytest.raises(RuntimeError, match="graph_preprocess"):
        prepare_attention(Graph(torch.tensor([0]), torch.tensor([1]), 2, 2))


def test_layers_pickled_without_an_attention():
    from tango_amd.gat import HGTLayer
    layer = HGTLayer(8, 8, 2)
    state = layer.__dict__.copy()
    for name in ("attention", "checkpoint"):
        del state[name]
    old = HGTLayer.__new__(HGTLayer)
    old.__setstate__(state)
    assert old.attention == "quantized" and old.checkpoint is None


def test_checkpoint_abi_refusals():
    from tango_amd import _lib
    L = _lib.lib()
    assert L.tango_pack_i8(16, 8, 16, 1, 1, 16, 3, 4, 8, 8, 8, None) == -2   # no such type
    assert L.tango_pack_i8(16, 8, 16, 1, 1, 16, 0, -1, 8, 8, 8, None) == -1
    assert L.tango_pack_i8(16, 8, 16, 1, 1, 16, 0, 4, 8, 8, 0, None) == -1   # group
    assert L.tango_pack_i8(16, 8, 16, 1, 1, None, 0, 4, 8, 8, 8, None) == -1
    assert L.tango_pack_i8(16, 4, 16, 1, 1, 16, 0, 4, 8, 8, 8, None) == -1   # rows of the result overlap
    assert L.tango_pack_i8(16, 8, 16, 1, 1, 18, 0, 4, 8, 8, 8, None) == -1   # fp32 off its alignment
    assert L.tango_pack_i8(16, 8, 16, 1, 1, 16, 0, 4, 1 << 30, 1 << 30, 8, None) == -2
    assert L.tango_pack_i8(None, 8, None, 1, 1, None, 0, 0, 8, 8, 8, None) == 0
    assert L.tango_pack_i8(16, 8, 16, -1, 1, 16, 0, 4, 8, 8, 8, None) == -1
    assert L.tango_unpack_i8(16, 0, 4, 16, 8, 16, 4, 8, 8, None) == -1
    assert L.tango_unpack_i8(16, 7, 8, 16, 8, 16, 4, 8, 8, None) == -2
    assert L.tango_unpack_i8(None, 0, 8, None, 8, None, 4, 0, 8, None) == 0


def test_weight_grad_abi_refusals():
    from tango_amd import _lib
    L = _lib.lib()
    ok = dict(dw=16, db=None, dy=16, dtype=0, ldy=8, q=16, ldq=16, scale=16, group=16, M=4, N=8, K=16, ws=None, nbytes=0, stream=None)
    call = lambda **kw: L.tango_weight_grad_i8(*{**ok, **kw}.values())
    assert call() == -4 and call(ws=16, nbytes=8) == -4
    assert call(dtype=5) == -2 and call(N=1 << 17) == -2 and call(M=1 << 31) == -2
    assert call(M=0) == -1 and call(group=0) == -1 and call(dy=None) == -1 and call(dw=18) == -1 and call(scale=None) == -1
    assert call(N=0) == 0 and call(K=0) == 0
    assert L.tango_weight_grad_i8_workspace(0, 4, 8, 16, 16) >= 4 * (8 * 16 + 8)
    assert L.tango_weight_grad_i8_workspace(0, 0, 8, 16, 16) == 0


def _attention(**kw):
    from tango_amd import _lib
    t = _lib.Attention(num_dst=4, num_src=4, heads=2, kv_heads=2, dim=8, q=16, k=16, v=16, q_row=16, q_head=8, k_row=16,
                       k_head=8, v_row=16, v_head=8, scale=1.0)
    i = _lib.AttnItems(num_items=4, num_edges=5, items=16, indices=16)
    for name, value in kw.items():
        setattr(i if hasattr(i, name) else t, name, value)
    return _lib.lib(), t, i


@pytest.mark.parametrize("status,change", [
    (-2, {"dtype": 3}), (-1, {"dim": 0}), (-2, {"dim": 257}), (-1, {"heads": 0}), (-2, {"heads": 3}), (-1, {"num_dst": -1}),
    (-2, {"num_src": 1 << 31}), (-1, {"q": None}), (-1, {"k": 18}), (-2, {"checkpoint": 1, "q_scale": 16, "k_scale": 16, "v_scale": 16}),
    (-1, {"checkpoint": 1}), (-1, {"num_items": 3}), (-1, {"items": 20}), (-1, {"indices": None}), (-2, {"num_edges": 1 << 31}),
    (-1, {"num_split": 1, "num_parts": 2, "split": None}), (-4, {"num_split": 1, "num_parts": 2, "split": 16}), (-1, {"num_src": 0}),
])
def test_attention_abi_refusals(status, change):
    L, t, i = _attention(**change)
    assert L.tango_graph_attention_fwd(16, ctypes.byref(t), ctypes.byref(i), None, None, 0, None) == status


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), 3e38, -3e38])
def test_attention_scale_out_of_range(scale):
    """Times log2(e), as the exponentials of base two take it, such a scale is not a finite fp32 number."""
    L, t, i = _attention(scale=scale)
    assert L.tango_graph_attention_fwd(16, ctypes.byref(t), ctypes.byref(i), None, None, 0, None) == -1
    assert L.tango_graph_attention_workspace(ctypes.byref(t), ctypes.byref(i), None, 1) == 0


def test_attention_backward_abi_refusals():
    L, t, i = _attention()
    refs = ctypes.byref(t), ctypes.byref(i)
    assert L.tango_graph_attention_bwd(16, 16, 16, refs[0], None, 16, 8, refs[1], refs[1], None, None, 0, None) == -1
    assert L.tango_graph_attention_bwd(16, 16, 16, refs[0], 16, 16, 8, refs[1], None, None, None, 0, None) == -1
    assert L.tango_graph_attention_bwd(16, 16, 16, refs[0], 16, 16, 8, refs[1], refs[1], None, None, 0, None) == -4
    assert L.tango_graph_attention_bwd(None, None, None, refs[0], 16, 16, 8, refs[1], refs[1], None, None, 0, None) == 0
    assert L.tango_graph_attention_fwd(None, refs[0], refs[1], None, None, 0, None) == -1
    assert L.tango_graph_attention_workspace(refs[0], refs[1], None, 0) == 0  # no row is cut
    assert L.tango_graph_attention_workspace(refs[0], refs[1], None, 1) >= 5 * 4
    assert L.tango_graph_attention_fwd(16, refs[0], refs[1], 16, None, 0, None) == -4
    assert L.tango_graph_attention_workspace(refs[0], refs[1], refs[1], 0) >= 4 * 2 * 8  # two floats a destination and head


def test_items_abi_refusals():
    from tango_amd import _lib
    L = _lib.lib()
    n = L.tango_attention_items_workspace()
    assert L.tango_attention_items(16, 16, 16, 4, 5, 0, 16, n, None) == -1
    assert L.tango_attention_items(16, 16, 16, 4, 5, 513, 16, n, None) == -2
    assert L.tango_attention_items(16, 16, 16, 1 << 31, 5, 8, 16, n, None) == -2
    assert L.tango_attention_items(16, 16, 16, 4, (1 << 30) + 1, 8, 16, n, None) == -2
    assert L.tango_attention_items(16, 16, 16, 4, 5, 8, 16, n - 1, None) == -4
    assert L.tango_attention_items(16, None, 16, 4, 9, 8, 16, n, None) == -1
    assert L.tango_attention_items(20, 16, 16, 4, 9, 8, 16, n, None) == -1
    assert L.tango_attention_items(None, None, None, 0, 0, 8, 16, n, None) == 0
