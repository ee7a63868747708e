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
from .checkpoint import DTYPES, need_float, on_device_of, pack_rows
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
    """One orientation of a graph cut into work items (``tango_attn_items`` of include/tango_hip.h)."""

    def __init__(self, indptr, indices, edge_ids, cap=None):
        cap = item_edges(indices.numel()) if cap is None else cap
        dev = indptr.device
        degree = indptr[1:] - indptr[:-1]
        rows = degree.numel()
        pieces = torch.clamp((degree + cap - 1) // cap, min=1)
        row = torch.repeat_interleave(torch.arange(rows, device=dev), pieces)
        nth = torch.arange(row.numel(), device=dev) - (torch.cumsum(pieces, 0) - pieces)[row]
        size = ((degree + pieces - 1) // pieces)[row]
        first = indptr[row] + nth * size
        last = torch.minimum(first + size, indptr[1:][row])
        cut = pieces[row] > 1
        part = torch.where(cut, torch.cumsum(cut, 0) - 1, -1)
        order = torch.sort(last - first, descending=True, stable=True).indices
        self.items = torch.stack([row, first, last, part], 1)[order].to(torch.int32).contiguous()
        split = torch.nonzero(pieces > 1).flatten()
        ends = torch.cumsum(pieces[split], 0)
        self.split = torch.stack([split, ends - pieces[split], ends, torch.zeros_like(split)], 1).to(torch.int32).contiguous()
        self.indices, self.edge_ids = indices, edge_ids
        s = _lib.AttnItems()
        s.num_items, s.num_split, s.num_edges = self.items.size(0), self.split.size(0), indices.numel()
        s.num_parts = int(ends[-1]) if ends.numel() else 0
        s.items, s.split, s.indices, s.edge_ids = _ptr(self.items), _ptr(self.split), _ptr(indices), _ptr(edge_ids)
        self.struct, self.ref = s, ctypes.byref(s)


def _items(graph, orientation):
    """The items of a preprocessed graph, built once per orientation and kept on the graph with the index arrays they
    were built from.  Building sorts on the device and reads counts back, so it cannot happen inside a capture."""
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
    torch.cuda.current_stream(indptr.device).synchronize()  # other streams may use the items from here on
    setattr(graph, "_attention_items_" + orientation, (indptr, narrow, items))
    return items


def prepare_attention(graph):
    """Builds what ``graph_attention`` keeps with a preprocessed graph (the first call does it otherwise); needed
    before a forward pass is captured into a HIP graph."""
    with on_device_of(graph.adj_csc[0]):
        _items(graph, "in")
        _items(graph, "out")
    return graph


def _unit_last(t):
    return t if t.dim() == 0 or t.size(-1) <= 1 or t.stride(-1) == 1 else t.contiguous()


def _struct(q_shape, k_shape, scale, dtype):
    t = _lib.Attention()
    t.num_dst, t.heads, t.dim = q_shape
    t.num_src, t.kv_heads = k_shape[:2]
    t.dtype, t.scale = DTYPES[dtype], scale
    return t


def _operands(t, q, k, v):
    t.q, t.k, t.v = _ptr(q), _ptr(k), _ptr(v)
    (t.q_row, t.q_head), (t.k_row, t.k_head), (t.v_row, t.v_head) = (x.stride()[:2] for x in (q, k, v))


def _hold(q, k, v):
    """8-bit values and scales of the three tensors, a scale per row and head.  The scales of a row's keys and values
    lie side by side, since the backward pass reads them together."""
    scales = [torch.empty(q.shape[:2] + (1,), dtype=torch.float32, device=q.device),
              torch.empty(k.shape[:2] + (2,), dtype=torch.float32, device=q.device)]
    flat = [x.reshape(x.size(0), x.size(1) * x.size(2)) for x in (q, k, v)]
    held = [pack_rows(x, q.size(2), s) for x, s in zip(flat, (scales[0][..., 0], scales[1][..., 0], scales[1][..., 1]))]
    return held, scales


def _checkpoint_operands(t, held, scales):
    t.checkpoint = 1
    for name, x in zip("qkv", held):
        setattr(t, name, _ptr(x))
        setattr(t, name + "_row", x.stride(0))
        setattr(t, name + "_head", t.dim)
    t.q_scale_row, t.q_scale_head = scales[0].stride()[:2]
    t.kv_scale_row, t.kv_scale_head = scales[1].stride()[:2]
    t.q_scale, t.k_scale = _ptr(scales[0]), _ptr(scales[1])
    t.v_scale = t.k_scale + 4 if t.k_scale else None


class _GraphAttention(Function):
    @staticmethod
    def forward(ctx, graph, q, k, v, scale, edge_mask, checkpoint):
        with on_device_of(q):
            by_dst = _items(graph, "in")
            q, k, v = _unit_last(q), _unit_last(k), _unit_last(v)
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
            t = _struct(q.shape, k.shape, scale, q.dtype)
            _operands(t, q, k, v)
            ref = ctypes.byref(t)
            ws_bytes = _L.tango_graph_attention_workspace(ref, by_dst.ref, None, edge_mask is not None)
            ws = _workspace(ws_bytes, q.device)
            check(_L.tango_graph_attention_fwd(_ptr(out), ref, by_dst.ref, _ptr(edge_mask), _ptr(ws), ws_bytes, _stream()),
                  "graph_attention")
            ctx.graph, ctx.scale, ctx.held = graph, scale, None
            if any(ctx.needs_input_grad[1:4]):
                if checkpoint:
                    ctx.held = _hold(q, k, v)
                    ctx.shapes = q.shape, k.shape, q.dtype
                    ctx.save_for_backward(edge_mask)
                else:
                    ctx.save_for_backward(edge_mask, q, k, v)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        refuse_capture("graph_attention.backward")
        with on_device_of(dout):
            by_dst, by_src = _items(ctx.graph, "in"), _items(ctx.graph, "out")
            edge_mask, *qkv = ctx.saved_tensors
            dout = _unit_last(dout)
            if ctx.held is None:
                q_shape, k_shape = qkv[0].shape, qkv[1].shape
                t = _struct(q_shape, k_shape, ctx.scale, qkv[0].dtype)
                _operands(t, *qkv)
            else:
                q_shape, k_shape, dtype = ctx.shapes
                t = _struct(q_shape, k_shape, ctx.scale, dtype)
                _checkpoint_operands(t, *ctx.held)
            grads = [torch.empty(shape, dtype=dout.dtype, device=dout.device) if need else None
                     for shape, need in zip((q_shape, k_shape, k_shape), ctx.needs_input_grad[1:4])]
            ref = ctypes.byref(t)
            ws_bytes = _L.tango_graph_attention_workspace(ref, by_dst.ref, by_src.ref, edge_mask is not None)
            ws = _workspace(ws_bytes, dout.device)
            check(_L.tango_graph_attention_bwd(*(None if g is None else _ptr(g) for g in grads), ref, _ptr(dout),
                                               dout.stride(0), dout.stride(1), by_dst.ref, by_src.ref, _ptr(edge_mask),
                                               _ptr(ws), ws_bytes, _stream()), "graph_attention.backward")
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
        if t.dtype != q.dtype or t.device != q.device:
            raise RuntimeError("graph_attention: q, k and v must have one type and one device")
    if not hasattr(graph, "adj_csc32"):
        raise RuntimeError("graph_attention: the graph has not been through graph_preprocess")
    num_dst, num_src = graph.adj_csc[0].numel() - 1, graph.adj_csr[0].numel() - 1
    if q.size(0) != num_dst or k.size(0) != num_src:
        raise RuntimeError("graph_attention: q needs a row per destination (%d), k and v one per source (%d)" % (num_dst, num_src))
    if k.shape != v.shape or q.size(2) != k.size(2):
        raise RuntimeError("graph_attention: k and v must have one shape, and q their dim")
    if not 1 <= q.size(2) <= 256:
        raise ValueError("graph_attention: dim must be 1 .. 256")
    if k.size(1) < 1 or q.size(1) % k.size(1) or q.size(1) < 1:
        raise ValueError("graph_attention: heads must be a multiple of kv_heads")
    if graph.adj_csc[0].device != q.device:
        raise RuntimeError("graph_attention: the graph and the tensors must be on one device")
    if edge_mask is not None:
        if not isinstance(edge_mask, torch.Tensor) or edge_mask.dtype != torch.bool or edge_mask.device != q.device:
            raise RuntimeError("graph_attention: edge_mask must be a bool tensor on q's device")
        if edge_mask.dim() != 1 or edge_mask.numel() != graph.adj_csc[1].numel():
            raise RuntimeError("graph_attention: edge_mask needs one entry per edge")
        edge_mask = edge_mask.contiguous()
    if checkpoint not in (None, "int8"):
        raise ValueError("graph_attention: checkpoint must be None or 'int8'")
    scale = 1.0 / math.sqrt(q.size(2)) if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError("graph_attention: scale must be finite")
    return _GraphAttention.apply(graph, q, k, v, scale, edge_mask, checkpoint == "int8")
