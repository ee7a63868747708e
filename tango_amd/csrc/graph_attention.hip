// C entries of the attention over a graph's edges: checks, workspace layout, the order of the passes.  The kernels are
// in graph_attention.hpp.
#include <math.h>

#include "graph_attention.hpp"

namespace tango {

extern template bool launch_attention<float, float>(AttnPass, AttnArgs, JoinArgs, int64_t, bool, hipStream_t);
extern template bool launch_attention<bf16_t, bf16_t>(AttnPass, AttnArgs, JoinArgs, int64_t, bool, hipStream_t);
extern template bool launch_attention<f16_t, f16_t>(AttnPass, AttnArgs, JoinArgs, int64_t, bool, hipStream_t);
extern template bool launch_attention<int8_t, float>(AttnPass, AttnArgs, JoinArgs, int64_t, bool, hipStream_t);
extern template bool launch_attention<int8_t, bf16_t>(AttnPass, AttnArgs, JoinArgs, int64_t, bool, hipStream_t);
extern template bool launch_attention<int8_t, f16_t>(AttnPass, AttnArgs, JoinArgs, int64_t, bool, hipStream_t);

static bool launch_any(const tango_attention& t, AttnPass pass, const AttnArgs& a, const JoinArgs& j, int64_t num_split,
                       bool aligned, hipStream_t s) {
    if (t.checkpoint) {
        if (t.dtype == TANGO_F32) return launch_attention<int8_t, float>(pass, a, j, num_split, aligned, s);
        if (t.dtype == TANGO_BF16) return launch_attention<int8_t, bf16_t>(pass, a, j, num_split, aligned, s);
        return launch_attention<int8_t, f16_t>(pass, a, j, num_split, aligned, s);
    }
    if (t.dtype == TANGO_F32) return launch_attention<float, float>(pass, a, j, num_split, aligned, s);
    if (t.dtype == TANGO_BF16) return launch_attention<bf16_t, bf16_t>(pass, a, j, num_split, aligned, s);
    return launch_attention<f16_t, f16_t>(pass, a, j, num_split, aligned, s);
}

static int check_shape(const tango_attention* t) {
    if (!t) return TANGO_ERR_INVALID_ARG;
    if (!float_type(t->dtype)) return TANGO_ERR_UNSUPPORTED;
    if (t->num_dst < 0 || t->num_src < 0 || t->heads <= 0 || t->kv_heads <= 0 || t->dim <= 0) return TANGO_ERR_INVALID_ARG;
    if (!(fabsf(t->scale) <= 0x1p127f)) return TANGO_ERR_INVALID_ARG;  // times log2(e) it has to be finite
    if (t->num_dst >= (1LL << 31) || t->num_src >= (1LL << 31) || t->heads > 65536 || t->heads % t->kv_heads || t->dim > 256)
        return TANGO_ERR_UNSUPPORTED;
    return TANGO_OK;
}

static int check_items(const tango_attn_items* i, int64_t rows) {
    if (!i || i->num_items < 0 || i->num_parts < 0 || i->num_split < 0 || i->num_edges < 0) return TANGO_ERR_INVALID_ARG;
    if (i->num_edges > (1LL << 30) || i->num_parts >= (1LL << 31)) return TANGO_ERR_UNSUPPORTED;
    if (i->num_items < rows || i->num_split > i->num_parts) return TANGO_ERR_INVALID_ARG;  // every row is at least one item
    if ((i->num_items && (!i->items || !aligned_to(i->items, 16))) || (i->num_split && (!i->split || !aligned_to(i->split, 16))))
        return TANGO_ERR_INVALID_ARG;
    if (i->num_edges && !i->indices) return TANGO_ERR_INVALID_ARG;
    return TANGO_OK;
}

static int64_t align256(int64_t b) { return (b + 255) & ~255LL; }

static int64_t masked_bytes(const tango_attn_items& i) { return align256(i.num_edges * 4); }
static int64_t forward_part_bytes(const tango_attention& t, const tango_attn_items& i) {
    return align256(i.num_parts * t.heads * (t.dim + 2) * 4);
}
// Whether the rows that a pass gathers from are more than the eight L2s of 4 MB hold.
static bool far_rows(int64_t rows, int64_t row_bytes) { return rows * row_bytes > (32LL << 20); }

static int64_t held_size(const tango_attention& t) { return t.checkpoint ? 1 : element_size(t.dtype); }

static bool keys_far(const tango_attention& t) { return far_rows(t.num_src, 2 * t.kv_heads * t.dim * held_size(t)); }
static bool queries_far(const tango_attention& t) {
    return far_rows(t.num_dst, t.heads * t.dim * (held_size(t) + element_size(t.dtype)));
}

static int query_tile_log(const tango_attention& t) {
    return head_tile_log(static_cast<int>(t.heads), static_cast<int>(t.heads / t.kv_heads), static_cast<int>(t.dim), held_size(t), 256);
}
static int key_tile_log(const tango_attention& t) {
    return head_tile_log(static_cast<int>(t.kv_heads), 1, static_cast<int>(t.dim), held_size(t), queries_far(t) ? 512 : 256);
}

// Query heads of a tile of the dk, dv pass; the statistics of the last tile are padded to as many.
static int stats_heads(const tango_attention& t) { return static_cast<int>(t.heads / t.kv_heads) << key_tile_log(t); }
static int64_t stats_bytes(const tango_attention& t) {
    return align256(ceil_div(t.heads, stats_heads(t)) * stats_heads(t) * t.num_dst * (t.checkpoint ? 16 : 8));
}
static int64_t backward_part_bytes(const tango_attention& t, const tango_attn_items& d, const tango_attn_items& s) {
    const int64_t a = align256(d.num_parts * t.heads * (2 * t.dim + 3) * 4), b = align256(s.num_parts * t.kv_heads * 2 * t.dim * 4);
    return a > b ? a : b;
}

static int check_operands(const tango_attention& t) {
    if ((t.num_dst && !t.q) || (t.num_src && (!t.k || !t.v))) return TANGO_ERR_INVALID_ARG;
    if (t.checkpoint && ((t.num_dst && !t.q_scale) || (t.num_src && (!t.k_scale || !t.v_scale)))) return TANGO_ERR_INVALID_ARG;
    const int64_t size = held_size(t);
    if (!aligned_to(t.q, size) || !aligned_to(t.k, size) || !aligned_to(t.v, size)) return TANGO_ERR_INVALID_ARG;
    return TANGO_OK;
}

// Whether a lane's pieces of `size`-byte elements can be loaded whole.
static bool rows_aligned(const void* p, int64_t row, int64_t head, int64_t vec, int64_t size) {
    const int64_t bytes = vec * size < 16 ? vec * size : 16;
    return aligned_to(p, bytes) && row * size % bytes == 0 && head * size % bytes == 0;
}

static void fill_args(AttnArgs& a, const tango_attention& t) {
    a = AttnArgs();
    a.q = t.q;
    a.k = t.k;
    a.v = t.v;
    a.q_scale = t.q_scale;
    a.k_scale = t.k_scale;
    a.v_scale = t.v_scale;
    a.q_row = t.q_row;
    a.q_head = t.q_head;
    a.k_row = t.k_row;
    a.k_head = t.k_head;
    a.v_row = t.v_row;
    a.v_head = t.v_head;
    a.heads = static_cast<int>(t.heads);
    a.kv_heads = static_cast<int>(t.kv_heads);
    a.rep = a.heads / a.kv_heads;
    a.dim = static_cast<int>(t.dim);
    a.scale = t.scale;
    a.num_dst = t.num_dst;
    a.qs_row = t.q_scale_row;
    a.qs_head = t.q_scale_head;
    a.kvs_row = t.kv_scale_row;
    a.kvs_head = t.kv_scale_head;
    a.stats_heads = stats_heads(t);
}

static void use_items(AttnArgs& a, JoinArgs& j, const tango_attn_items& i, const uint8_t* mask, int32_t* masked, int tile_log, bool far,
                      hipStream_t s) {
    a.items = reinterpret_cast<const int4*>(i.items);
    a.num_items = i.num_items;
    a.indices = i.indices;
    if (mask && i.num_edges) {
        hipLaunchKernelGGL(attn_mask_kernel, dim3(grid_for(i.num_edges, 256)), dim3(256), 0, s, masked, i.indices, i.edge_ids, mask,
                           static_cast<uint32_t>(i.num_edges));
        a.indices = masked;
    }
    a.tile_log = tile_log;
    a.tile_slow = far;
    j.split = reinterpret_cast<const int4*>(i.split);
    j.parts = a.parts;
    j.out = a.out;
    j.out2 = a.out2;
    j.stats = a.stats;
    j.q_scale = a.q_scale;
    j.num_dst = a.num_dst;
    j.qs_row = a.qs_row;
    j.qs_head = a.qs_head;
    j.stats_heads = a.stats_heads;
    j.dim = a.dim;
    j.scale = a.scale;
}

// ---- Work items.  A row of d edges is ceil(d / cap) pieces (one if d is 0) of ceil(d / pieces) edges, the last one
// shorter; items are counted by length, the counts become the first places of the lengths, longest first, and the pieces
// take places.  Which of equal lengths comes first depends on the order of the workgroups, what is computed from the
// items does not: an item owns its row or a numbered part of it.

constexpr int kLengths = 513;  // 0 .. 512 edges

struct ItemCounts {
    int32_t split, parts;
    int32_t place[kLengths];  // items of a length, then the next place of one
};

struct RowPieces {
    int64_t first;
    int degree, pieces, size, last;  // pieces - 1 of `size` edges and one of `last`
};

__device__ __forceinline__ RowPieces row_pieces(const int64_t* indptr, int64_t row, int cap) {
    RowPieces p;
    p.first = indptr[row];
    p.degree = static_cast<int>(indptr[row + 1] - p.first);
    p.pieces = p.degree > cap ? (p.degree + cap - 1) / cap : 1;
    p.size = (p.degree + p.pieces - 1) / p.pieces;
    p.last = p.degree - (p.pieces - 1) * p.size;
    return p;
}

static __global__ __launch_bounds__(256) void items_count_kernel(ItemCounts* c, const int64_t* indptr, int64_t rows, int cap) {
    __shared__ int32_t count[kLengths];
    for (int i = threadIdx.x; i < kLengths; i += 256) count[i] = 0;
    __syncthreads();
    const int64_t row = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (row < rows) {
        const RowPieces p = row_pieces(indptr, row, cap);
        if (p.pieces > 1) atomicAdd(&count[p.size], p.pieces - 1);
        atomicAdd(&count[p.last], 1);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kLengths; i += 256)
        if (count[i]) atomicAdd(&c->place[i], count[i]);
}

static __global__ __launch_bounds__(64) void items_scan_kernel(ItemCounts* c) {
    if (threadIdx.x) return;
    int32_t at = 0;
    for (int i = kLengths - 1; i >= 0; --i) {
        const int32_t n = c->place[i];
        c->place[i] = at;
        at += n;
    }
}

static __global__ __launch_bounds__(256) void items_place_kernel(int4* items, int4* split, ItemCounts* c, const int64_t* indptr,
                                                                 int64_t rows, int cap) {
    __shared__ int32_t count[kLengths], base[kLengths];
    for (int i = threadIdx.x; i < kLengths; i += 256) count[i] = 0;
    __syncthreads();
    const int64_t row = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const bool on = row < rows;
    RowPieces p = {0, 0, 1, 0, 0};
    int32_t full_at = 0, last_at = 0;
    if (on) {
        p = row_pieces(indptr, row, cap);
        if (p.pieces > 1) full_at = atomicAdd(&count[p.size], p.pieces - 1);
        last_at = atomicAdd(&count[p.last], 1);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kLengths; i += 256)
        if (count[i]) base[i] = atomicAdd(&c->place[i], count[i]);
    __syncthreads();
    if (!on) return;
    const int r = static_cast<int>(row), first = static_cast<int>(p.first);
    int part = -1;
    if (p.pieces > 1) {
        part = atomicAdd(&c->parts, p.pieces);
        split[atomicAdd(&c->split, 1)] = make_int4(r, part, part + p.pieces, 0);
        full_at += base[p.size];
        for (int i = 0; i + 1 < p.pieces; ++i)
            items[full_at + i] = make_int4(r, first + i * p.size, first + (i + 1) * p.size, part + i);
    }
    items[base[p.last] + last_at] =
        make_int4(r, first + p.degree - p.last, first + p.degree, p.pieces > 1 ? part + p.pieces - 1 : -1);
}

}  // namespace tango

using namespace tango;

extern "C" {

size_t tango_attention_items_workspace(void) { return sizeof(ItemCounts); }

int tango_attention_items(int32_t* items, int32_t* split, const int64_t* indptr, int64_t rows, int64_t num_edges, int64_t cap,
                          void* counts, size_t counts_bytes, tango_stream_t stream) {
    if (rows < 0 || num_edges < 0 || cap < 1) return TANGO_ERR_INVALID_ARG;
    if (cap >= kLengths || rows >= (1LL << 31) || num_edges > (1LL << 30) || rows + num_edges / cap >= (1LL << 31))
        return TANGO_ERR_UNSUPPORTED;
    if (!counts || counts_bytes < sizeof(ItemCounts) || !aligned_to(counts, 16)) return TANGO_ERR_WORKSPACE;
    if (rows == 0) return TANGO_OK;
    if (!items || !indptr || !aligned_to(items, 16) || !aligned_to(split, 16) || (num_edges > cap && !split)) return TANGO_ERR_INVALID_ARG;
    ItemCounts* c = static_cast<ItemCounts*>(counts);
    const dim3 grid(static_cast<uint32_t>(ceil_div(rows, 256))), block(256);
    hipStream_t s = as_stream(stream);
    hipLaunchKernelGGL(items_count_kernel, grid, block, 0, s, c, indptr, rows, static_cast<int>(cap));
    hipLaunchKernelGGL(items_scan_kernel, dim3(1), dim3(64), 0, s, c);
    hipLaunchKernelGGL(items_place_kernel, grid, block, 0, s, reinterpret_cast<int4*>(items), reinterpret_cast<int4*>(split), c, indptr,
                       rows, static_cast<int>(cap));
    return launch_status();
}

size_t tango_graph_attention_workspace(const tango_attention* t, const tango_attn_items* by_dst, const tango_attn_items* by_src,
                                       int masked) {
    if (check_shape(t) != TANGO_OK || !by_dst) return 0;
    const int64_t mask = masked ? masked_bytes(*by_dst) : 0;
    if (!by_src) return static_cast<size_t>(mask + forward_part_bytes(*t, *by_dst));
    return static_cast<size_t>(mask + stats_bytes(*t) + backward_part_bytes(*t, *by_dst, *by_src));
}

int tango_graph_attention_fwd(void* out, const tango_attention* t, const tango_attn_items* by_dst, const uint8_t* edge_mask,
                              void* workspace, size_t workspace_bytes, tango_stream_t stream) {
    int rc = check_shape(t);
    if (rc == TANGO_OK) rc = check_items(by_dst, t->num_dst);
    if (rc == TANGO_OK) rc = check_operands(*t);
    if (rc != TANGO_OK) return rc;
    if (t->checkpoint) return TANGO_ERR_UNSUPPORTED;  // the forward pass runs on the tensors themselves
    if (t->num_dst == 0) return TANGO_OK;
    if (!out || (by_dst->num_edges && t->num_src == 0)) return TANGO_ERR_INVALID_ARG;
    const int64_t mask_bytes = edge_mask ? masked_bytes(*by_dst) : 0;
    const int64_t need = mask_bytes + forward_part_bytes(*t, *by_dst);
    if (need && (!workspace || static_cast<int64_t>(workspace_bytes) < need || !aligned_to(workspace, 16))) return TANGO_ERR_WORKSPACE;
    AttnArgs a;
    JoinArgs j = JoinArgs();
    fill_args(a, *t);
    a.out = out;
    int32_t* masked = static_cast<int32_t*>(workspace);
    a.parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + mask_bytes);
    const int64_t size = element_size(t->dtype), vec = attention_vec(size);
    use_items(a, j, *by_dst, edge_mask, masked, query_tile_log(*t), keys_far(*t), as_stream(stream));
    const bool aligned = t->dim % vec == 0 && rows_aligned(t->q, t->q_row, t->q_head, vec, size) &&
                         rows_aligned(t->k, t->k_row, t->k_head, vec, size) && rows_aligned(t->v, t->v_row, t->v_head, vec, size) &&
                         aligned_to(out, 16);
    if (!launch_any(*t, kPassForward, a, j, by_dst->num_split, aligned, as_stream(stream))) return TANGO_ERR_UNSUPPORTED;
    return launch_status();
}

int tango_graph_attention_bwd(void* dq, void* dk, void* dv, const tango_attention* t, const void* dout, int64_t dout_row,
                              int64_t dout_head, const tango_attn_items* by_dst, const tango_attn_items* by_src,
                              const uint8_t* edge_mask, void* workspace, size_t workspace_bytes, tango_stream_t stream) {
    int rc = check_shape(t);
    if (rc == TANGO_OK) rc = check_items(by_dst, t->num_dst);
    if (rc == TANGO_OK) rc = check_items(by_src, t->num_src);
    if (rc == TANGO_OK) rc = check_operands(*t);
    if (rc != TANGO_OK) return rc;
    if (by_dst->num_edges != by_src->num_edges || (t->num_dst && !dout)) return TANGO_ERR_INVALID_ARG;
    if (by_dst->num_edges && (t->num_src == 0 || t->num_dst == 0)) return TANGO_ERR_INVALID_ARG;
    if (!dq && !dk && !dv) return TANGO_OK;
    const int64_t mask_bytes = edge_mask ? masked_bytes(*by_dst) : 0;
    const int64_t need = mask_bytes + stats_bytes(*t) + backward_part_bytes(*t, *by_dst, *by_src);
    if (need && (!workspace || static_cast<int64_t>(workspace_bytes) < need || !aligned_to(workspace, 16))) return TANGO_ERR_WORKSPACE;
    const int64_t size = t->checkpoint ? 1 : element_size(t->dtype), vec = attention_vec(size);
    const int64_t gsize = element_size(t->dtype);
    const bool aligned = t->dim % vec == 0 && rows_aligned(t->q, t->q_row, t->q_head, vec, size) &&
                         rows_aligned(t->k, t->k_row, t->k_head, vec, size) && rows_aligned(t->v, t->v_row, t->v_head, vec, size) &&
                         rows_aligned(dout, dout_row, dout_head, vec, gsize) && aligned_to(dq, 16) && aligned_to(dk, 16) &&
                         aligned_to(dv, 16);
    AttnArgs a;
    JoinArgs j = JoinArgs();
    fill_args(a, *t);
    a.dout = dout;
    a.do_row = dout_row;
    a.do_head = dout_head;
    int32_t* masked = static_cast<int32_t*>(workspace);
    a.stats = reinterpret_cast<float*>(static_cast<char*>(workspace) + mask_bytes);
    a.parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + mask_bytes + stats_bytes(*t));
    if (t->num_dst) {
        a.out = dq;
        use_items(a, j, *by_dst, edge_mask, masked, query_tile_log(*t), keys_far(*t), as_stream(stream));
        if (!launch_any(*t, kPassQuery, a, j, by_dst->num_split, aligned, as_stream(stream))) return TANGO_ERR_UNSUPPORTED;
        rc = launch_status();
        if (rc != TANGO_OK) return rc;
    }
    if (t->num_src && (dk || dv)) {
        a.out = dk;
        a.out2 = dv;
        use_items(a, j, *by_src, edge_mask, masked, key_tile_log(*t), queries_far(*t), as_stream(stream));
        if (!launch_any(*t, kPassKeyValue, a, j, by_src->num_split, aligned, as_stream(stream))) return TANGO_ERR_UNSUPPORTED;
        rc = launch_status();
    }
    return rc;
}

}  // extern "C"
