// Softmax attention over the edges of a graph: out[d, h] = sum over the in-edges e = (s -> d) of p_e v[s, h'] with
// p = softmax over those edges of scale * (q[d, h] . k[s, h']), h' = h / (heads / kv_heads); and its gradient, which
// keeps nothing per edge and forms the probabilities again.
//
//   forward   one pass over a destination's edges with the running maximum m and sum l of its softmax: a step of U
//             edges raises m to the largest of their logits, scales l and the running sum of v by 2^(m_old - m_new)
//             and adds the U terms.  Logits are held times log2(e), so that exp is one v_exp_f32.
//   dq        with dp_e = dout[d] . v[s], delta = sum p dp:  dq[d] = scale sum_e p_e (dp_e - delta) k[s].  One pass over
//             the destination's edges as well: beside m and l it carries sum p dp, A = sum p dp k and B = sum p k, and
//             ends with dq = scale (A - delta B) / l.  Neither the output nor anything else of the forward pass is
//             needed, and delta carries no rounding of a stored 16-bit output.  The pass leaves log2 of the
//             softmax's denominator and delta of each (destination, head) for the next one.
//   dk, dv    one pass over a source's out-edges: p = 2^(logit - log2 denominator), dv[s] += p dout[d],
//             dk[s] += scale p (dp - delta) q[d]; over all query heads that share the key head.
//
// Work items.  A row (destination or source) with its edges is cut into items of at most 16 .. 512 edges; items are
// sorted by length, longest first, so that the items of a wavefront end together and the launch has no long tail.  A
// row that is one item is finished by its owner; rows of several items leave partial results that a join kernel adds
// in item order: no result depends on scheduling, and no sum is made with atomics.
//
// Lanes.  An item and a tile of heads belong to G lanes: LPH lanes for each head, VEC elements (16 bytes of the
// gathered type) each, and as many neighbouring heads as bring the gathered piece of a row to 256 bytes, two lines of L2
// (fp32 [169343, 8, 32] with 1.3 M edges: forward 390 us, 395 us with 128 bytes, 404 us with 512).  The dk, dv pass takes
// 512 bytes unless all it gathers from fits the L2s: a line of statistics goes with each piece of a row (at
// [232965, 8, 32] bf16 and 9.4 M edges 1440 us, 1570 us with 256 bytes, 1740 us with 128; at 19717 rows and 0.2 M edges
// 31 us against 28 us with 256).
//
// What bounds the passes: two gathered rows an edge, most of them from beyond L2 (no graph order is assumed); the
// fabric behind the L2s delivers 7 to 8 TB/s.  Order of the workgroups: if the rows that a pass gathers from are more
// than the L2s hold together, the head tile varies slowest, so that all XCDs gather from the same columns and these
// stay in the 256 MB cache in front of the memory (forward at 169343 rows of 8 x 32 fp32: 390 us against 415 us); if
// they fit, it varies fastest, so that an XCD's L2 sees the columns of its own tiles only (19717 rows of 8 x 32 bf16:
// 25 us against 31 us).
#pragma once
#include "element.hpp"

namespace tango {

constexpr float kLog2e = 1.4426950408889634f;

struct AttnArgs {
    const void *q, *k, *v, *dout;
    const float *q_scale, *k_scale, *v_scale;  // int8 operands: one scale per (row, head), at row * .._row + head * .._head
    int64_t qs_row, qs_head, kvs_row, kvs_head;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, do_row, do_head;  // strides in elements
    void *out, *out2;  // [rows, heads, dim] contiguous
    float* stats;      // per tile of the dk, dv pass [destinations, query heads of the tile]: an AttnStat
    int64_t num_dst;
    int stats_heads;   // query heads of such a tile
    float* parts;      // partial results of rows of several items
    const int4* items; // row, first slot, last slot + 1, part or -1
    const int32_t* indices;  // the other endpoint of a slot's edge; negative: the edge takes no part
    int64_t num_items;
    int heads, kv_heads, rep, dim, tiles, tile_log;
    int tile_slow;  // the head tile varies slowest over the workgroups, not fastest
    float scale;
};

template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}

// Sum over LPH neighbouring lanes, in all of them (the mirror steps pair lanes whose halves already hold equal sums).
template <int LPH>
__device__ __forceinline__ float lanes_sum(float x) {
    if constexpr (LPH >= 2) x += dpp<0xb1>(x);    // quad_perm 1 0 3 2
    if constexpr (LPH >= 4) x += dpp<0x4e>(x);    // quad_perm 2 3 0 1
    if constexpr (LPH >= 8) x += dpp<0x141>(x);   // row_half_mirror
    if constexpr (LPH >= 16) x += dpp<0x140>(x);  // row_mirror
    if constexpr (LPH >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    if constexpr (LPH >= 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return x;
}

// How a lane reaches its VEC elements of a head's row (the lanes of a head are numbered j = 0 .. LPH - 1).
//   kWhole    dim is a multiple of VEC and every row starts on a vector: elements j VEC .. j VEC + VEC - 1.
//   kShifted  any dim >= VEC, any alignment: the same, except that the last lane with elements is moved back to end with
//             the row, so that every load is one whole vector inside the row.  What it then shares with its neighbour
//             is masked to zero.  (dim 250 in fp16, [169343, 3, 250] and 1.3 M edges: forward 746 us instead of 1800 us with
//             a load per element.)
//   kSingle   dim < VEC: one lane, a load per element.
enum RowMode { kWhole, kShifted, kSingle };

template <int VEC, int LPH, int MODE>
struct RowLane {
    int start, first, dim;  // first element held; the first of them that is this lane's (VEC: none)
    __device__ __forceinline__ RowLane(int j, int d) : dim(d) {
        if constexpr (MODE == kWhole) {
            start = j * VEC;
            first = start < d ? 0 : VEC;
        } else if constexpr (MODE == kShifted) {
            start = j * VEC < d - VEC ? j * VEC : d - VEC;
            first = j * VEC < d ? j * VEC - start : VEC;
        } else {
            start = first = 0;
        }
    }
    __device__ __forceinline__ bool mine(int i) const { return MODE == kSingle ? i < dim : i >= first; }
};

template <typename T, int VEC, int LPH, int MODE>
struct HeadRow {
    Pack<T, VEC> p;
    __device__ __forceinline__ void zero() { p.zero(); }
    // the words are zero before
    __device__ __forceinline__ void load(const T* head, const RowLane<VEC, LPH, MODE>& lane) {
        constexpr int kBits = 8 * static_cast<int>(sizeof(T));
        if constexpr (MODE == kWhole) {
            if (lane.first == 0) p.load(head + lane.start);
        } else if constexpr (MODE == kShifted) {
            p.load_any(head + lane.start);
            const int cut = lane.first * kBits;  // bits from the front on that are the neighbour's
#pragma unroll
            for (int i = 0; i < Pack<T, VEC>::kWords; ++i) {
                const int c = cut - 32 * i;
                p.w[i] &= c <= 0 ? 0xffffffffu : c >= 32 ? 0u : 0xffffffffu << (c & 31);
            }
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (i < lane.dim) {
                    Pack<T, 1> one;
                    one.load(head + i);
                    p.w[i * kBits / 32] |= one.w[0] << (i * kBits % 32);
                }
        }
    }
    __device__ __forceinline__ float get(int i) const { return p.get(i); }
};

template <typename T, int VEC, int LPH, int MODE>
__device__ __forceinline__ void store_head(T* head, const RowLane<VEC, LPH, MODE>& lane, const float* v) {
    if (MODE != kSingle && lane.first == 0) {
        Pack<T, VEC> o;
        o.set_all(v);
        if constexpr (MODE == kWhole) o.store(head + lane.start);
        if constexpr (MODE == kShifted) o.store_any(head + lane.start);
        return;
    }
    if (MODE == kWhole) return;
#pragma unroll
    for (int i = 0; i < VEC; ++i)
        if (lane.mine(i)) {
            Pack<T, 1> o;
            o.set_all(v + i);
            o.store(head + lane.start + i);
        }
}

template <int VEC, int LPH, int MODE>
__device__ __forceinline__ void store_part(float* head, const RowLane<VEC, LPH, MODE>& lane, const float* v) {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
        if (lane.mine(i)) head[lane.start + i] = v[i];
}

struct ItemLane {
    int4 it;  // row, first slot, last slot + 1, part
    int head, j;
    bool on;  // a real item and a real head
};

template <int LPH>
__device__ __forceinline__ ItemLane item_lane(const AttnArgs& a, int heads) {
    ItemLane r;
    const int g_log = a.tile_log + __builtin_ctz(LPH);
    const int gl = threadIdx.x & ((1 << g_log) - 1);
    const uint32_t inner = a.tile_slow ? gridDim.x / static_cast<uint32_t>(a.tiles) : static_cast<uint32_t>(a.tiles);
    const uint32_t outer_id = blockIdx.x / inner, inner_id = blockIdx.x - outer_id * inner;
    const int64_t block = a.tile_slow ? inner_id : outer_id;
    const int tile = static_cast<int>(a.tile_slow ? outer_id : inner_id);
    const int64_t id = block * (256 >> g_log) + (threadIdx.x >> g_log);
    r.head = (tile << a.tile_log) + gl / LPH;
    r.j = gl & (LPH - 1);
    r.on = id < a.num_items && r.head < heads;
    r.it = r.on ? a.items[id] : make_int4(0, 0, 0, -1);
    return r;
}

// U slots from e on: their row ids, and whether they take part.
template <int U>
struct Slots {
    int32_t id[U];
    bool ok[U];
    __device__ __forceinline__ void load(const AttnArgs& a, int e, int end) {
#pragma unroll
        for (int u = 0; u < U; ++u) id[u] = a.indices[e + u < end ? e + u : end - 1];
#pragma unroll
        for (int u = 0; u < U; ++u) ok[u] = e + u < end;
    }
    __device__ __forceinline__ bool take(int u) const { return ok[u] && id[u] >= 0; }
};

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// 2^(m_old - m_new) for running maxima, with 1 for -inf against -inf
__device__ __forceinline__ float rescale(float m_old, float m_new) { return m_old == m_new ? 1.0f : exp2_fast(m_old - m_new); }

// The maximum to subtract: 0 while no finite logit has been seen, so that 2^(-inf - m) is 0 and not NaN.
__device__ __forceinline__ float shift_of(float m) { return m == -INFINITY ? 0.0f : m; }

// log2 of the softmax's denominator; +inf for a destination that nothing is left of, so that 2^(logit - it) is 0
__device__ __forceinline__ float log2_total(float m, float l) { return l == 0.0f ? INFINITY : m + __builtin_amdgcn_logf(l); }

// Edges of a step (rows of both gathered tensors are in flight together; more cost registers and so wavefronts).
// Forward at 2 / 4 / 6 / 8: 424 / 413 / 391 / 387 us ([169343, 8, 32] fp32, 1.3 M edges), 577 / 552 / 553 / 605 us (5.3 M
// edges, heads 8 over 2).  dq: 456 / 430 / 425 / 422 us, from checkpoints [169343, 4, 64] 197 / 225 / 235 / 213 us;
// dk, dv: 489 / 486 / 492 / 541 us, from checkpoints 310 / 315 / 351 / 532 us.
// Rows that no vector divides take four forward: the masks of six cost more registers ([169343, 3, 250] fp16: 730 us
// against 790 us).
constexpr int forward_edges(int mode) { return mode == kWhole ? 6 : 4; }
constexpr int backward_edges(bool scaled) { return scaled ? 2 : 4; }

template <typename T, int VEC, int LPH, int MODE>
__global__ __launch_bounds__(256) void attn_fwd_kernel(const AttnArgs a) {
    constexpr int U = forward_edges(MODE);
    const ItemLane L = item_lane<LPH>(a, a.heads);
    if (!L.on) return;
    const RowLane<VEC, LPH, MODE> lane(L.j, a.dim);
    const int kvh = L.head / a.rep;
    const T* k = static_cast<const T*>(a.k) + kvh * a.k_head;
    const T* v = static_cast<const T*>(a.v) + kvh * a.v_head;
    float q[VEC], acc[VEC];
    {
        HeadRow<T, VEC, LPH, MODE> r;
        r.zero();
        r.load(static_cast<const T*>(a.q) + L.it.x * a.q_row + L.head * a.q_head, lane);
        const float f = a.scale * kLog2e;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            q[i] = r.get(i) * f;
            acc[i] = 0.0f;
        }
    }
    float m = -INFINITY, l = 0.0f;
    const int end = L.it.z;
    Slots<U> cur, next;
    if (L.it.y < end) next.load(a, L.it.y, end);
    for (int e = L.it.y; e < end; e += U) {
        cur = next;
#pragma unroll
        for (int u = 0; u < U; ++u) cur.ok[u] = cur.take(u);
        HeadRow<T, VEC, LPH, MODE> kr[U], vr[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            kr[u].zero();
            if (cur.ok[u]) kr[u].load(k + cur.id[u] * a.k_row, lane);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            vr[u].zero();
            if (cur.ok[u]) vr[u].load(v + cur.id[u] * a.v_row, lane);
        }
        if (e + U < end) next.load(a, e + U, end);
        float s[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float t = 0.0f;
#pragma unroll
            for (int i = 0; i < VEC; ++i) t = __builtin_fmaf(q[i], kr[u].get(i), t);
            t = lanes_sum<LPH>(t);
            s[u] = cur.ok[u] ? t : -INFINITY;
        }
        float m_new = m;
#pragma unroll
        for (int u = 0; u < U; ++u) m_new = fmaxf(m_new, s[u]);
        const float shift = shift_of(m_new), c = rescale(m, m_new);
        m = m_new;
        l *= c;
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] *= c;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float p = exp2_fast(s[u] - shift);
            l += p;
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[i] = __builtin_fmaf(p, vr[u].get(i), acc[i]);
        }
    }
    if (L.it.w < 0) {
        const float r = l == 0.0f ? 0.0f : 1.0f / l;  // a destination that nothing is left of gets zeros
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] *= r;
        T* out = static_cast<T*>(a.out) + (static_cast<int64_t>(L.it.x) * a.heads + L.head) * a.dim;
        store_head<T, VEC, LPH, MODE>(out, lane, acc);
    } else {
        float* part = a.parts + (static_cast<int64_t>(L.it.w) * a.heads + L.head) * (a.dim + 2);
        if (L.j == 0) {
            part[0] = m;
            part[1] = l;
        }
        store_part<VEC, LPH, MODE>(part + 2, lane, acc);
    }
}

template <typename T>
struct RowScale {
    static constexpr bool kScaled = __is_same(T, int8_t);
    static __device__ __forceinline__ float get(const float* scale, int64_t row, int64_t row_step, int64_t head) {
        if constexpr (kScaled) return scale[row * row_step + head];
        return 1.0f;
    }
};

// What the dk, dv pass needs of a (destination, query head) beside its rows: log2 of the softmax's denominator, delta, and
// from checkpoints the query's scale.  Laid out so that what a lane group reads of a destination is contiguous: with
// all heads of a destination together, a tile of one head would fetch a line for 8 bytes of it (at [169343, 8, 32] fp32
// and 1.3 M edges that pass took 690 us, 610 us with the tile's alone).
template <bool SCALED>
struct AttnStat {
    static constexpr int kFloats = SCALED ? 4 : 2;
    static __device__ __forceinline__ void store(float* stats, int64_t num_dst, int per_tile, int64_t row, int head, float total,
                                                 float delta, float scale) {
        const int tile = head / per_tile;
        float* p = stats + ((tile * num_dst + row) * per_tile + (head - tile * per_tile)) * kFloats;
        if constexpr (SCALED)
            *reinterpret_cast<float4*>(p) = make_float4(total, delta, scale, 0.0f);
        else
            *reinterpret_cast<float2*>(p) = make_float2(total, delta);
    }
    static __device__ __forceinline__ float4 load(const float* tile, int64_t at) {
        if constexpr (SCALED) return *reinterpret_cast<const float4*>(tile + at * 4);
        const float2 t = *reinterpret_cast<const float2*>(tile + at * 2);
        return make_float4(t.x, t.y, 1.0f, 0.0f);
    }
};

// T: what q, k, v are held in (int8_t: checkpoints, with a scale per row and head); TG: dout and the results
template <typename T, typename TG, int VEC, int LPH, int MODE>
__global__ __launch_bounds__(256) void attn_bwd_q_kernel(const AttnArgs a) {
    typedef RowScale<T> S;
    constexpr int U = backward_edges(S::kScaled);
    const ItemLane L = item_lane<LPH>(a, a.heads);
    if (!L.on) return;
    const RowLane<VEC, LPH, MODE> lane(L.j, a.dim);
    const int kvh = L.head / a.rep;
    const T* k = static_cast<const T*>(a.k) + kvh * a.k_head;
    const T* v = static_cast<const T*>(a.v) + kvh * a.v_head;
    const float qs = S::get(a.q_scale, L.it.x, a.qs_row, L.head * a.qs_head);
    float q[VEC], g[VEC], A[VEC], B[VEC];
    {
        HeadRow<T, VEC, LPH, MODE> r;
        HeadRow<TG, VEC, LPH, MODE> o;
        r.zero();
        o.zero();
        r.load(static_cast<const T*>(a.q) + L.it.x * a.q_row + L.head * a.q_head, lane);
        o.load(static_cast<const TG*>(a.dout) + L.it.x * a.do_row + L.head * a.do_head, lane);
        const float f = qs * a.scale * kLog2e;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            q[i] = r.get(i) * f;
            g[i] = o.get(i);
            A[i] = B[i] = 0.0f;
        }
    }
    float m = -INFINITY, l = 0.0f, dsum = 0.0f;
    const int end = L.it.z;
    Slots<U> cur, next;
    if (L.it.y < end) next.load(a, L.it.y, end);
    for (int e = L.it.y; e < end; e += U) {
        cur = next;
#pragma unroll
        for (int u = 0; u < U; ++u) cur.ok[u] = cur.take(u);
        HeadRow<T, VEC, LPH, MODE> kr[U], vr[U];
        float ks[U], vs[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            kr[u].zero();
            vr[u].zero();
            ks[u] = vs[u] = 1.0f;
            if (cur.ok[u]) {
                kr[u].load(k + cur.id[u] * a.k_row, lane);
                vr[u].load(v + cur.id[u] * a.v_row, lane);
                ks[u] = S::get(a.k_scale, cur.id[u], a.kvs_row, kvh * a.kvs_head);
                vs[u] = S::get(a.v_scale, cur.id[u], a.kvs_row, kvh * a.kvs_head);
            }
        }
        if (e + U < end) next.load(a, e + U, end);
        float s[U], dp[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float t = 0.0f, w = 0.0f;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                t = __builtin_fmaf(q[i], kr[u].get(i), t);
                w = __builtin_fmaf(g[i], vr[u].get(i), w);
            }
            t = lanes_sum<LPH>(t);
            w = lanes_sum<LPH>(w);
            if constexpr (S::kScaled) {
                t *= ks[u];
                w *= vs[u];
            }
            s[u] = cur.ok[u] ? t : -INFINITY;
            dp[u] = cur.ok[u] ? w : 0.0f;
        }
        float m_new = m;
#pragma unroll
        for (int u = 0; u < U; ++u) m_new = fmaxf(m_new, s[u]);
        const float shift = shift_of(m_new), c = rescale(m, m_new);
        m = m_new;
        l *= c;
        dsum *= c;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            A[i] *= c;
            B[i] *= c;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float p = exp2_fast(s[u] - shift);
            const float pd = p * dp[u];
            l += p;
            dsum += pd;
            const float pb = S::kScaled ? p * ks[u] : p, pa = S::kScaled ? pd * ks[u] : pd;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                A[i] = __builtin_fmaf(pa, kr[u].get(i), A[i]);
                B[i] = __builtin_fmaf(pb, kr[u].get(i), B[i]);
            }
        }
    }
    if (L.it.w < 0) {
        const float r = l == 0.0f ? 0.0f : 1.0f / l;
        const float delta = dsum * r;
        const float f = a.scale * r;
#pragma unroll
        for (int i = 0; i < VEC; ++i) A[i] = (A[i] - delta * B[i]) * f;
        const int64_t at = static_cast<int64_t>(L.it.x) * a.heads + L.head;
        if (a.out) store_head<TG, VEC, LPH, MODE>(static_cast<TG*>(a.out) + at * a.dim, lane, A);
        if (L.j == 0) AttnStat<S::kScaled>::store(a.stats, a.num_dst, a.stats_heads, L.it.x, L.head, log2_total(m, l), delta, qs);
    } else {
        float* part = a.parts + (static_cast<int64_t>(L.it.w) * a.heads + L.head) * (2 * a.dim + 3);
        if (L.j == 0) {
            part[0] = m;
            part[1] = l;
            part[2] = dsum;
        }
        store_part<VEC, LPH, MODE>(part + 3, lane, A);
        store_part<VEC, LPH, MODE>(part + 3 + a.dim, lane, B);
    }
}

template <typename T, typename TG, int VEC, int LPH, int MODE>
__global__ __launch_bounds__(256) void attn_bwd_kv_kernel(const AttnArgs a) {
    typedef RowScale<T> S;
    constexpr int U = backward_edges(S::kScaled);
    const ItemLane L = item_lane<LPH>(a, a.kv_heads);
    if (!L.on) return;
    const RowLane<VEC, LPH, MODE> lane(L.j, a.dim);
    const T* q = static_cast<const T*>(a.q) + static_cast<int64_t>(L.head) * a.rep * a.q_head;
    const TG* o = static_cast<const TG*>(a.dout) + static_cast<int64_t>(L.head) * a.rep * a.do_head;
    const int in_tile = L.head & ((1 << a.tile_log) - 1);
    const float* stats = a.stats + ((L.head >> a.tile_log) * a.num_dst * a.stats_heads + in_tile * a.rep) * AttnStat<S::kScaled>::kFloats;
    float k[VEC], v[VEC], dk[VEC], dv[VEC];
    {
        HeadRow<T, VEC, LPH, MODE> kr, vr;
        kr.zero();
        vr.zero();
        kr.load(static_cast<const T*>(a.k) + L.it.x * a.k_row + L.head * a.k_head, lane);
        vr.load(static_cast<const T*>(a.v) + L.it.x * a.v_row + L.head * a.v_head, lane);
        const float f = S::get(a.k_scale, L.it.x, a.kvs_row, L.head * a.kvs_head) * a.scale * kLog2e;
        const float fv = S::get(a.v_scale, L.it.x, a.kvs_row, L.head * a.kvs_head);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            k[i] = kr.get(i) * f;
            v[i] = vr.get(i) * fv;
            dk[i] = dv[i] = 0.0f;
        }
    }
    const int end = L.it.z;
    Slots<U> cur, next;
    if (L.it.y < end) next.load(a, L.it.y, end);
    for (int e = L.it.y; e < end; e += U) {
        cur = next;
#pragma unroll
        for (int u = 0; u < U; ++u) cur.ok[u] = cur.take(u);
        if (e + U < end) next.load(a, e + U, end);
        for (int r = 0; r < a.rep; ++r) {
            HeadRow<T, VEC, LPH, MODE> qr[U];
            HeadRow<TG, VEC, LPH, MODE> gr[U];
            float4 st[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                qr[u].zero();
                gr[u].zero();
                st[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (cur.ok[u]) {
                    qr[u].load(q + cur.id[u] * a.q_row + r * a.q_head, lane);
                    gr[u].load(o + cur.id[u] * a.do_row + r * a.do_head, lane);
                    st[u] = AttnStat<S::kScaled>::load(stats, static_cast<int64_t>(cur.id[u]) * a.stats_heads + r);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float t = 0.0f, w = 0.0f;
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    t = __builtin_fmaf(k[i], qr[u].get(i), t);
                    w = __builtin_fmaf(v[i], gr[u].get(i), w);
                }
                t = lanes_sum<LPH>(t);
                w = lanes_sum<LPH>(w);
                if constexpr (S::kScaled) t *= st[u].z;
                const float p = cur.ok[u] ? exp2_fast(t - st[u].x) : 0.0f;
                float ds = cur.ok[u] ? p * (w - st[u].y) : 0.0f;
                if constexpr (S::kScaled) ds *= st[u].z;
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    dk[i] = __builtin_fmaf(ds, qr[u].get(i), dk[i]);
                    dv[i] = __builtin_fmaf(p, gr[u].get(i), dv[i]);
                }
            }
        }
    }
    if (L.it.w < 0) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) dk[i] *= a.scale;
        const int64_t at = (static_cast<int64_t>(L.it.x) * a.kv_heads + L.head) * a.dim;
        if (a.out) store_head<TG, VEC, LPH, MODE>(static_cast<TG*>(a.out) + at, lane, dk);
        if (a.out2) store_head<TG, VEC, LPH, MODE>(static_cast<TG*>(a.out2) + at, lane, dv);
    } else {
        float* part = a.parts + (static_cast<int64_t>(L.it.w) * a.kv_heads + L.head) * (2 * a.dim);
        store_part<VEC, LPH, MODE>(part, lane, dk);
        store_part<VEC, LPH, MODE>(part + a.dim, lane, dv);
    }
}

// Joins the parts of a row of several items.  A workgroup owns 64 of the row's heads * dim elements, one a lane; each of
// its four waves takes every fourth part, and the four running results are added in order.
struct JoinArgs {
    const int4* split;  // row, first part, last part + 1
    const float* parts;
    void *out, *out2;
    float* stats;
    const float* q_scale;
    int64_t num_dst, qs_row, qs_head;
    int stats_heads, heads, dim, windows;
    float scale;
};

enum JoinKind { kJoinForward, kJoinQuery, kJoinKeyValue };

template <typename T, int KIND, bool SCALED>
__global__ __launch_bounds__(256) void attn_join_kernel(const JoinArgs a) {
    constexpr int kHead = KIND == kJoinForward ? 2 : KIND == kJoinQuery ? 3 : 0;
    __shared__ float sm[4][64], sl[4][64], sd[4][64], sx[4][64], sy[4][64];
    const uint32_t row_id = blockIdx.x / static_cast<uint32_t>(a.windows);
    const int4 sp = a.split[row_id];
    const int lane = threadIdx.x & 63, slice = threadIdx.x >> 6;
    const int e = static_cast<int>(blockIdx.x - row_id * a.windows) * 64 + lane;
    const bool on = e < a.heads * a.dim;
    const int head = on ? e / a.dim : 0, d = on ? e - head * a.dim : 0;
    const int len = (KIND == kJoinForward ? 1 : 2) * a.dim + kHead;
    const int64_t step = static_cast<int64_t>(len) * a.heads;
    const float* p = a.parts + sp.y * step + static_cast<int64_t>(head) * len;
    const int n = sp.z - sp.y;
    float m = -INFINITY, l = 0.0f, dsum = 0.0f, x = 0.0f, y = 0.0f;
#pragma unroll 4
    for (int i = slice; i < n; i += 4) {
        const float* r = p + i * step;
        const float px = r[kHead + d], py = KIND == kJoinForward ? 0.0f : r[kHead + a.dim + d];
        if constexpr (KIND == kJoinKeyValue) {
            x += px;
            y += py;
        } else {
            const float pm = r[0], m_new = fmaxf(m, pm);
            const float c = rescale(m, m_new), pc = exp2_fast(pm - shift_of(m_new));
            m = m_new;
            l = __builtin_fmaf(r[1], pc, l * c);
            x = __builtin_fmaf(px, pc, x * c);
            if constexpr (KIND == kJoinQuery) {
                dsum = __builtin_fmaf(r[2], pc, dsum * c);
                y = __builtin_fmaf(py, pc, y * c);
            }
        }
    }
    sx[slice][lane] = x;
    if constexpr (KIND != kJoinForward) sy[slice][lane] = y;
    if constexpr (KIND != kJoinKeyValue) {
        sm[slice][lane] = m;
        sl[slice][lane] = l;
    }
    if constexpr (KIND == kJoinQuery) sd[slice][lane] = dsum;
    __syncthreads();
    if (slice != 0 || !on) return;
    if constexpr (KIND != kJoinKeyValue) m = fmaxf(fmaxf(sm[0][lane], sm[1][lane]), fmaxf(sm[2][lane], sm[3][lane]));
    l = dsum = x = y = 0.0f;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const float c = KIND == kJoinKeyValue ? 1.0f : exp2_fast(sm[s][lane] - shift_of(m));
        x = __builtin_fmaf(sx[s][lane], c, x);
        if constexpr (KIND != kJoinForward) y = __builtin_fmaf(sy[s][lane], c, y);
        if constexpr (KIND != kJoinKeyValue) l = __builtin_fmaf(sl[s][lane], c, l);
        if constexpr (KIND == kJoinQuery) dsum = __builtin_fmaf(sd[s][lane], c, dsum);
    }
    const int64_t at = (static_cast<int64_t>(sp.x) * a.heads + head) * a.dim + d;
    const float r = l == 0.0f ? 0.0f : 1.0f / l;
    if constexpr (KIND == kJoinForward) {
        static_cast<T*>(a.out)[at] = static_cast<T>(x * r);
    } else if constexpr (KIND == kJoinQuery) {
        const float delta = dsum * r;
        if (a.out) static_cast<T*>(a.out)[at] = static_cast<T>((x - delta * y) * (a.scale * r));
        if (d == 0)
            AttnStat<SCALED>::store(a.stats, a.num_dst, a.stats_heads, sp.x, head, log2_total(m, l), delta,
                                    SCALED ? a.q_scale[sp.x * a.qs_row + head * a.qs_head] : 1.0f);
    } else {
        if (a.out) static_cast<T*>(a.out)[at] = static_cast<T>(x * a.scale);
        if (a.out2) static_cast<T*>(a.out2)[at] = static_cast<T>(y);
    }
}

// indices with the edges that a mask leaves out made negative: the passes then read one number a slot, not a chain of
// three (slot, edge id, mask) in front of every gather (forward at 5.3 M edges, heads 8 over 2,
// fp32: 1040 us with the chain, 550 us and 45 us for this kernel without)
static __global__ __launch_bounds__(256) void attn_mask_kernel(int32_t* out, const int32_t* indices, const int32_t* edge_ids,
                                                               const uint8_t* mask, uint32_t n) {
    const uint32_t stride = gridDim.x * 256;
    for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < n; i += stride)
        out[i] = mask[edge_ids ? static_cast<uint32_t>(edge_ids[i]) : i] ? indices[i] : -1;
}

enum AttnPass { kPassForward, kPassQuery, kPassKeyValue };

// Launches one pass over `items` and its join; `aligned`: rows are reached by vector loads.  T: fp32 / bf16 / fp16
// operands, or int8_t checkpoints under results of type TG.  False: a grid beyond the device's limit.
template <typename T, typename TG>
bool launch_attention(AttnPass pass, AttnArgs a, JoinArgs j, int64_t num_split, bool aligned, hipStream_t s);

// Lanes of a head: a power of two with a vector of VEC elements each.
inline int head_lanes_log(int dim, int vec) {
    int log = 0;
    while ((vec << log) < dim) ++log;
    return log;
}

// Elements per lane: 16 bytes of fp32, bf16, fp16; 8 of int8 (whose gradients are four or two times as wide).
inline int attention_vec(int64_t size) { return size == 4 ? 4 : 8; }

// Neighbouring heads of a lane group, as a power of two: what brings the gathered piece of a row to `bytes`.  Query heads
// that share a key head count once: their lanes read the same addresses.
inline int head_tile_log(int heads, int rep, int dim, int64_t size, int64_t bytes) {
    const int vec = attention_vec(size), lanes = static_cast<int>(bytes / (vec * size));
    const int lph_log = head_lanes_log(dim, vec);
    int log = 0;
    while ((1 << (lph_log + log)) < lanes * rep && (1 << (lph_log + log)) < kWave && (1 << log) < heads) ++log;
    return log;
}

template <typename T, typename TG, int VEC, int LPH, int MODE>
bool launch_attention_lanes(AttnPass pass, AttnArgs& a, hipStream_t s) {
    const int64_t per_block = 256 / (LPH << a.tile_log);
    const int64_t blocks = ceil_div(a.num_items, per_block) * a.tiles;
    if (blocks > 0x7fffffffLL) return false;
    if (blocks == 0) return true;
    const dim3 grid(static_cast<uint32_t>(blocks)), block(256);
    if (pass == kPassForward) {
        if constexpr (__is_same(T, TG)) hipLaunchKernelGGL((attn_fwd_kernel<T, VEC, LPH, MODE>), grid, block, 0, s, a);
    } else if (pass == kPassQuery) {
        hipLaunchKernelGGL((attn_bwd_q_kernel<T, TG, VEC, LPH, MODE>), grid, block, 0, s, a);
    } else {
        hipLaunchKernelGGL((attn_bwd_kv_kernel<T, TG, VEC, LPH, MODE>), grid, block, 0, s, a);
    }
    return true;
}

template <typename T, typename TG, int VEC, int MODE>
bool launch_attention_vec(AttnPass pass, AttnArgs& a, hipStream_t s) {
    switch (head_lanes_log(a.dim, VEC)) {
        case 0: return launch_attention_lanes<T, TG, VEC, 1, MODE>(pass, a, s);
        case 1: return launch_attention_lanes<T, TG, VEC, 2, MODE>(pass, a, s);
        case 2: return launch_attention_lanes<T, TG, VEC, 4, MODE>(pass, a, s);
        case 3: return launch_attention_lanes<T, TG, VEC, 8, MODE>(pass, a, s);
        case 4: return launch_attention_lanes<T, TG, VEC, 16, MODE>(pass, a, s);
        case 5: return launch_attention_lanes<T, TG, VEC, 32, MODE>(pass, a, s);
        case 6:
            if constexpr (VEC == 4) return launch_attention_lanes<T, TG, VEC, 64, MODE>(pass, a, s);
    }
    return false;
}

template <typename T, typename TG>
bool launch_attention(AttnPass pass, AttnArgs a, JoinArgs j, int64_t num_split, bool aligned, hipStream_t s) {
    constexpr int VEC = sizeof(T) == 4 ? 4 : 8;
    constexpr bool kScaled = RowScale<T>::kScaled;
    const int heads = pass == kPassKeyValue ? a.kv_heads : a.heads;
    a.tiles = static_cast<int>(ceil_div(heads, 1 << a.tile_log));
    const bool ok = a.dim < VEC ? launch_attention_lanes<T, TG, VEC, 1, kSingle>(pass, a, s)
                    : aligned   ? launch_attention_vec<T, TG, VEC, kWhole>(pass, a, s)
                                : launch_attention_vec<T, TG, VEC, kShifted>(pass, a, s);
    if (!ok) return false;
    if (num_split == 0) return true;
    j.heads = heads;
    j.windows = static_cast<int>(ceil_div(static_cast<int64_t>(heads) * a.dim, 64));
    const int64_t blocks = num_split * j.windows;
    if (blocks > 0x7fffffffLL) return false;
    const dim3 grid(static_cast<uint32_t>(blocks)), block(256);
    if (pass == kPassForward)
        hipLaunchKernelGGL((attn_join_kernel<TG, kJoinForward, kScaled>), grid, block, 0, s, j);
    else if (pass == kPassQuery)
        hipLaunchKernelGGL((attn_join_kernel<TG, kJoinQuery, kScaled>), grid, block, 0, s, j);
    else
        hipLaunchKernelGGL((attn_join_kernel<TG, kJoinKeyValue, kScaled>), grid, block, 0, s, j);
    return true;
}

}  // namespace tango
