"""Multi-head softmax attention over a graph's edges in one pass each way, with nothing kept per edge.

The reference's attention layers run a dot SDDMM, DGL's edge softmax and a weighted SpMM with an [E, heads] tensor
between them (evaluation/test_HGT.py:52-62), and the quantized operators here do the same in int8.  ``graph_attention``
is that chain on the floating-point tensors themselves: a running maximum and sum per destination and head instead of
stored logits, and a backward pass that forms the probabilities again, from q, k and v or from their 8-bit
checkpoints."""
import ctypes
import math

import torch
from torch.autograd.function import Function, once_differentiable

from . import _lib
from .checkpoint import DTYPES, need_float, on_device_of, pack_rows, rows_of
from .kernels import _L, _ptr, _stream, _workspace, check, refuse_capture


def item_edges(edges):
    """Edges of a work item at most, by the graph's size: the power of two from sqrt(edges) / 16 on, 16 .. 512.  Short
    items end together and let a small graph fill the device; long ones leave less to join (forward and join in us at
    caps 16 / 32 / 64 / 128 / 256: 4.1 k edges 10 / 12 / 16 / 24 / 35, 0.2 M 35 / 29 / 29 / 44 / 73, 1.3 M 447 / 416 /
    410 / 401 / 415, 9.4 M 1918 / 1479 / 1311 / 1261 / 1235)."""
    cap = 16
    while cap < 512 and 256 * cap * cap < edges:
        cap *= 2
    return cap


class AttentionItems:
    """One orientation of a graph cut into work items (``tango_attn_items`` of include/tango_hip.h) on its device."""

    def __init__(self, indptr, indices, edge_ids, cap=None):
        cap = item_edges(indices.numel()) if cap is None else cap
        device, rows, edges = indptr.device, indptr.numel() - 1, indices.numel()
        items = torch.empty((rows + edges // cap, 4), dtype=torch.int32, device=device)
        split = torch.empty((edges // cap, 4), dtype=torch.int32, device=device)
        nbytes = _L.tango_attention_items_workspace()
        counts = torch.zeros(nbytes // 4, dtype=torch.int32, device=device)
        check(_L.tango_attention_items(_ptr(items), _ptr(split), _ptr(indptr), rows, edges, cap, _ptr(counts), nbytes, _stream()),
              "attention_items")
        num_split, num_parts = counts[:2].tolist()  # waits for the kernels: any stream may use the items from here on
        self.items, self.split = items[:rows - num_split + num_parts], split[:num_split]
        self.indices, self.edge_ids, self.num_parts = indices, edge_ids, num_parts
        self._point()

    def _point(self):
        s = _lib.AttnItems()
        s.num_items, s.num_split, s.num_parts, s.num_edges = self.items.size(0), self.split.size(0), self.num_parts, self.indices.numel()
        s.items, s.split, s.indices, s.edge_ids = _ptr(self.items), _ptr(self.split), _ptr(self.indices), _ptr(self.edge_ids)
        self.struct, self.ref = s, ctypes.byref(s)

    def __getstate__(self):
        """A graph is copied and saved with its items: without the addresses, which are the copy's own."""
        return {name: value for name, value in self.__dict__.items() if name not in ("struct", "ref")}

    def __setstate__(self, state):
        self.__dict__.update(state)
        self._point()


def _items(graph, orientation):
    """The items of a preprocessed graph, built once per orientation and kept on the graph with the index arrays they
    were built from.  Building reads two counts back, so it cannot happen inside a capture."""
    fmt, narrow, ordered = (("adj_csc", "adj_csc32", "csc_slots_are_edge_ids") if orientation == "in" else
                            ("adj_csr", "adj_csr32", "csr_slots_are_edge_ids"))
    if not hasattr(graph, narrow):
        raise RuntimeError("graph_attention: the graph has not been through graph_preprocess")
    indptr, narrow = getattr(graph, fmt)[0], getattr(graph, narrow)
    kept = getattr(graph, "_attention_items_" + orientation, None)
    if kept is not None and kept[0] is indptr and kept[1] is narrow:
        return kept[2]
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("graph_attention: run prepare_attention(graph) before capturing")
    items = AttentionItems(indptr, narrow[0], None if getattr(graph, ordered) else narrow[1])
    setattr(graph, "_attention_items_" + orientation, (indptr, narrow, items))
    return items


def prepare_attention(graph):
    """Builds what ``graph_attention`` keeps with a preprocessed graph (the first call does it otherwise); needed
    before a forward pass is captured into a HIP graph."""
    if not hasattr(graph, "adj_csc32"):
        raise RuntimeError("graph_attention: the graph has not been through graph_preprocess")
    with on_device_of(graph.adj_csc[0]):
        _items(graph, "in")
        _items(graph, "out")
    return graph


def _unit_last(t):
    return t if t.size(-1) <= 1 or t.stride(-1) == 1 else t.contiguous()


def _hold(q, k, v):
    """8-bit values and scales of the three tensors, a scale per row and head.  The scales of a row's keys and values
    lie side by side, since the backward pass reads them together."""
    scales = [torch.empty(q.shape[:2] + (1,), dtype=torch.float32, device=q.device),
              torch.empty(k.shape[:2] + (2,), dtype=torch.float32, device=q.device)]
    # heads of one column may lie apart: those are copied, as all are that no view makes rows of
    flat = [x.view(x.size(0), x.size(1) * x.size(2)) if x.is_contiguous() else rows_of(x.flatten(1)) for x in (q, k, v)]
    held = [pack_rows(x, q.size(2), s) for x, s in zip(flat, (scales[0][..., 0], scales[1][..., 0], scales[1][..., 1]))]
    return (*held, *scales)


def _struct(q, k, v, scale):
    """tango_attention of the tensors themselves."""
    n, heads, dim = q.shape
    (qr, qh, _), (kr, kh, _), (vr, vh, _) = q.stride(), k.stride(), v.stride()
    return _lib.Attention(n, k.size(0), heads, k.size(1), dim, DTYPES[q.dtype], 0, _ptr(q), _ptr(k), _ptr(v), qr, qh, kr, kh, vr, vh,
                          None, None, None, 0, 0, 0, 0, scale)


def _struct_held(q_shape, k_shape, dtype, q, k, v, q_scale, kv_scale, scale):
    """tango_attention of their 8-bit forms."""
    (n, heads, dim), (m, kv_heads, _) = q_shape, k_shape
    at = _ptr(kv_scale)
    return _lib.Attention(n, m, heads, kv_heads, dim, DTYPES[dtype], 1, _ptr(q), _ptr(k), _ptr(v), q.stride(0), dim, k.stride(0), dim,
                          v.stride(0), dim, _ptr(q_scale), at, at + 4 if at else None, *q_scale.stride()[:2],
                          *kv_scale.stride()[:2], scale)


class _GraphAttention(Function):
    @staticmethod
    def forward(ctx, graph, q, k, v, scale, edge_mask, checkpoint):
        with on_device_of(q):
            by_dst = _items(graph, "in")
            q, k, v = _unit_last(q), _unit_last(k), _unit_last(v)
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
            ref = ctypes.byref(_struct(q, k, v, scale))
            ws_bytes = _L.tango_graph_attention_workspace(ref, by_dst.ref, None, edge_mask is not None)
            ws = _workspace(ws_bytes, q.device)
            check(_L.tango_graph_attention_fwd(_ptr(out), ref, by_dst.ref, _ptr(edge_mask), _ptr(ws), ws_bytes, _stream()),
                  "graph_attention")
            ctx.graph, ctx.scale, ctx.held = graph, scale, None
            if any(ctx.needs_input_grad[1:4]):
                if checkpoint:
                    ctx.held = q.shape, k.shape, q.dtype
                    ctx.save_for_backward(edge_mask, *_hold(q, k, v))
                else:
                    ctx.save_for_backward(edge_mask, q, k, v)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        refuse_capture("graph_attention.backward")
        with on_device_of(dout):
            by_dst, by_src = _items(ctx.graph, "in"), _items(ctx.graph, "out")
            edge_mask, *kept = ctx.saved_tensors
            dout = _unit_last(dout)
            if ctx.held is None:
                t = _struct(*kept, ctx.scale)
                q_shape, k_shape = kept[0].shape, kept[1].shape
            else:
                q_shape, k_shape, dtype = ctx.held
                t = _struct_held(q_shape, k_shape, dtype, *kept, ctx.scale)
            grads = [torch.empty(shape, dtype=dout.dtype, device=dout.device) if need else None
                     for shape, need in zip((q_shape, k_shape, k_shape), ctx.needs_input_grad[1:4])]
            ref = ctypes.byref(t)
            ws_bytes = _L.tango_graph_attention_workspace(ref, by_dst.ref, by_src.ref, edge_mask is not None)
            ws = _workspace(ws_bytes, dout.device)
            check(_L.tango_graph_attention_bwd(*map(_ptr, grads), ref, _ptr(dout), dout.stride(0), dout.stride(1), by_dst.ref,
                                               by_src.ref, _ptr(edge_mask), _ptr(ws), ws_bytes, _stream()),
                  "graph_attention.backward")
        return None, grads[0], grads[1], grads[2], None, None, None


def graph_attention(graph, q, k, v, scale=None, edge_mask=None, checkpoint=None):
    """``out[d, h] = sum over the in-edges e = (s -> d) of softmax_e(scale * q[d, h] . k[s, h']) v[s, h']``.

    ``q`` [destinations, heads, dim], ``k`` and ``v`` [sources, kv_heads, dim], one type (fp32, bf16 or fp16), heads a
    multiple of kv_heads (head h reads key head h' = h // (heads / kv_heads)), dim <= 256; any strides with contiguous
    columns are read in place.  ``graph``: preprocessed (``graph_preprocess``), square or bipartite.  ``scale``:
    default 1 / sqrt(dim).  ``edge_mask``: bool [edges] by edge id, False = the edge takes no part, whatever its key and
    value hold.  A destination that no edge is left of gets zeros and passes no gradient on.
    ``checkpoint="int8"``: what the backward pass needs of q, k and v is kept in 8 bits with a scale per row and head
    (``tango_amd.checkpoint.pack``); the output is the same, the gradients are the attention's at the held values.
    Sums, softmax statistics and the partial results of long rows are fp32; outputs and gradients are rounded once."""
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        need_float(t, name)
        if t.dim() != 3:
            raise RuntimeError("graph_attention: %s must be [nodes, heads, dim]" % name)
    if not (q.dtype == k.dtype == v.dtype and q.device == k.device == v.device):
        raise RuntimeError("graph_attention: q, k and v must have one type and one device")
    if not hasattr(graph, "adj_csc32"):
        raise RuntimeError("graph_attention: the graph has not been through graph_preprocess")
    by_dst = graph.adj_csc[0]
    num_dst, num_src = by_dst.size(0) - 1, graph.adj_csr[0].size(0) - 1
    (rows, heads, dim), (k_rows, kv_heads, k_dim) = q.shape, k.shape
    if rows != num_dst or k_rows != num_src:
        raise RuntimeError("graph_attention: q needs a row per destination (%d), k and v one per source (%d)" % (num_dst, num_src))
    if k.shape != v.shape or k_dim != dim:
        raise RuntimeError("graph_attention: k and v must have one shape, and q their dim")
    if not 1 <= dim <= 256:
        raise ValueError("graph_attention: dim must be 1 .. 256")
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError("graph_attention: heads must be a multiple of kv_heads")
    if by_dst.device != q.device:
        raise RuntimeError("graph_attention: the graph and the tensors must be on one device")
    if edge_mask is not None:
        if not isinstance(edge_mask, torch.Tensor) or edge_mask.dtype != torch.bool or edge_mask.device != q.device:
            raise RuntimeError("graph_attention: edge_mask must be a bool tensor on q's device")
        if edge_mask.dim() != 1 or edge_mask.numel() != graph.adj_csc[1].numel():
            raise RuntimeError("graph_attention: edge_mask needs one entry per edge")
        edge_mask = edge_mask.contiguous()
    if checkpoint not in (None, "int8"):
        raise ValueError("graph_attention: checkpoint must be None or 'int8'")
    scale = 1.0 / math.sqrt(dim) if scale is None else float(scale)
    if not abs(scale) <= 2.0 ** 127:  # times log2(e) it has to be finite in fp32
        raise ValueError("graph_attention: scale must be finite, 2^127 at most")
    return _GraphAttention.apply(graph, q, k, v, scale, edge_mask, checkpoint == "int8")
