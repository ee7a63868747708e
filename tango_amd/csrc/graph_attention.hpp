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
// Work items.  A row (destination or source) with its edges is cut into items of at most kItemEdges edges; items are
// sorted by length, longest first, so that the items of a wavefront end together and the launch has no long tail.  A
// row that is one item is finished by its owner; rows of several items leave partial results that a join kernel adds
// in item order: nothing here depends on scheduling, and there are no atomics.
//
// Lanes.  An item and a tile of heads belong to G lanes: LPH lanes for each head, VEC elements (16 bytes of the
// gathered type) each, and as many neighbouring heads as bring the gathered piece of a row to 128 bytes, the line
// of L2.  The head tile varies fastest over the workgroups: consecutive workgroups go to different XCDs, so an L2
// sees the key and value columns of few heads (with eight tiles: of one).
#pragma once
#include "element.hpp"

namespace tango {

constexpr float kLog2e = 1.4426950408889634f;

struct AttnArgs {
    const void *q, *k, *v, *dout;
    const float *q_scale, *k_scale, *v_scale;  // int8 operands: one scale per (row, head)
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, do_row, do_head;  // strides in elements
    void *out, *out2;  // [rows, heads, dim] contiguous
    float2* stats;     // [destinations, heads]: log2 of the softmax's denominator, delta
    float* parts;      // partial results of rows of several items
    const int4* items; // row, first slot, last slot + 1, part or -1
    const int32_t* indices;
    const int32_t* edge_ids;  // NULL: a slot's number is its edge's
    const uint8_t* mask;      // by edge id; NULL: every edge takes part
    int64_t num_items;
    int heads, kv_heads, rep, dim, tiles, tile_log;
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

// A lane's VEC elements of one head's row.  AL: consecutive elements in vector loads (VEC divides dim and every row
// start is aligned); else elements lane, lane + LPH, ... one load each.
template <typename T, int VEC, int LPH, bool AL>
struct HeadRow {
    Pack<T, VEC> p;
    __device__ __forceinline__ void zero() { p.zero(); }
    __device__ __forceinline__ void load(const T* head, int j, int dim) {
        if constexpr (AL) {
            if (j * VEC < dim) p.load(head + j * VEC);
        } else {
            constexpr int kBits = 8 * static_cast<int>(sizeof(T));
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const int c = i * LPH + j;
                if (c < dim) {
                    Pack<T, 1> one;
                    one.load(head + c);
                    p.w[i * kBits / 32] |= one.w[0] << (i * kBits % 32);  // the words are zero before
                }
            }
        }
    }
    __device__ __forceinline__ float get(int i) const { return p.get(i); }
};

template <typename T, int VEC, int LPH, bool AL>
__device__ __forceinline__ void store_head(T* head, int j, int dim, const float* v) {
    if constexpr (AL) {
        if (j * VEC < dim) {
            Pack<T, VEC> o;
            o.set_all(v);
            o.store(head + j * VEC);
        }
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const int c = i * LPH + j;
            if (c < dim) {
                Pack<T, 1> o;
                o.set_all(v + i);
                o.store(head + c);
            }
        }
    }
}

template <int VEC, int LPH, bool AL>
__device__ __forceinline__ void store_part(float* head, int j, int dim, const float* v) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        const int c = AL ? j * VEC + i : i * LPH + j;
        if (c < dim) head[c] = v[i];
    }
}

struct ItemLane {
    int4 it;  // row, first slot, last slot + 1, part
    int head, j;
    bool item, on;  // a real item; and a real head
};

template <int LPH>
__device__ __forceinline__ ItemLane item_lane(const AttnArgs& a, int heads) {
    ItemLane r;
    const int g_log = a.tile_log + __builtin_ctz(LPH);
    const int gl = threadIdx.x & ((1 << g_log) - 1);
    const int64_t block = blockIdx.x / static_cast<uint32_t>(a.tiles);
    const int tile = static_cast<int>(blockIdx.x - static_cast<uint32_t>(block) * a.tiles);
    const int64_t id = block * (256 >> g_log) + (threadIdx.x >> g_log);
    r.head = (tile << a.tile_log) + gl / LPH;
    r.j = gl & (LPH - 1);
    r.item = id < a.num_items;
    r.on = r.item && r.head < heads;
    r.it = r.item ? a.items[id] : make_int4(0, 0, 0, -1);
    return r;
}

// U slots from e on: their row ids, and whether they take part.
template <int U>
struct Slots {
    int32_t id[U];
    bool ok[U];
    __device__ __forceinline__ void load(const AttnArgs& a, int e, int end) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            ok[u] = e + u < end;
            id[u] = a.indices[ok[u] ? e + u : end - 1];
        }
        if (a.mask) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int slot = ok[u] ? e + u : end - 1;
                ok[u] = ok[u] && a.mask[a.edge_ids ? a.edge_ids[slot] : slot];
            }
        }
    }
};

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// 2^(m_old - m_new) for running maxima, with 1 for -inf against -inf
__device__ __forceinline__ float rescale(float m_old, float m_new) { return m_old == m_new ? 1.0f : exp2_fast(m_old - m_new); }

// The maximum to subtract: 0 while no finite logit has been seen, so that 2^(-inf - m) is 0 and not NaN.
__device__ __forceinline__ float shift_of(float m) { return m == -INFINITY ? 0.0f : m; }

// log2 of the softmax's denominator; +inf for a destination that nothing is left of, so that 2^(logit - it) is 0
__device__ __forceinline__ float log2_total(float m, float l) { return l == 0.0f ? INFINITY : m + __builtin_amdgcn_logf(l); }

constexpr int kEdgesInFlight = 4;

template <typename T, int VEC, int LPH, bool AL>
__global__ __launch_bounds__(256) void attn_fwd_kernel(const AttnArgs a) {
    constexpr int U = kEdgesInFlight;
    const ItemLane L = item_lane<LPH>(a, a.heads);
    if (!L.on) return;
    const int kvh = L.head / a.rep;
    const T* k = static_cast<const T*>(a.k) + kvh * a.k_head;
    const T* v = static_cast<const T*>(a.v) + kvh * a.v_head;
    float q[VEC], acc[VEC];
    {
        HeadRow<T, VEC, LPH, AL> r;
        r.zero();
        r.load(static_cast<const T*>(a.q) + L.it.x * a.q_row + L.head * a.q_head, L.j, a.dim);
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
        HeadRow<T, VEC, LPH, AL> kr[U], vr[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            kr[u].zero();
            if (cur.ok[u]) kr[u].load(k + cur.id[u] * a.k_row, L.j, a.dim);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            vr[u].zero();
            if (cur.ok[u]) vr[u].load(v + cur.id[u] * a.v_row, L.j, a.dim);
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
        store_head<T, VEC, LPH, AL>(out, L.j, a.dim, acc);
    } else {
        float* part = a.parts + (static_cast<int64_t>(L.it.w) * a.heads + L.head) * (a.dim + 2);
        if (L.j == 0) {
            part[0] = m;
            part[1] = l;
        }
        store_part<VEC, LPH, AL>(part + 2, L.j, a.dim, acc);
    }
}

template <typename T>
struct RowScale {
    static constexpr bool kScaled = __is_same(T, int8_t);
    static __device__ __forceinline__ float get(const float* scale, int64_t row, int heads, int head) {
        if constexpr (kScaled) return scale[row * heads + head];
        return 1.0f;
    }
};

// T: what q, k, v are held in (int8_t: checkpoints, with a scale per row and head); TG: dout and the results
template <typename T, typename TG, int VEC, int LPH, bool AL>
__global__ __launch_bounds__(256) void attn_bwd_q_kernel(const AttnArgs a) {
    constexpr int U = kEdgesInFlight;
    typedef RowScale<T> S;
    const ItemLane L = item_lane<LPH>(a, a.heads);
    if (!L.on) return;
    const int kvh = L.head / a.rep;
    const T* k = static_cast<const T*>(a.k) + kvh * a.k_head;
    const T* v = static_cast<const T*>(a.v) + kvh * a.v_head;
    float q[VEC], g[VEC], A[VEC], B[VEC];
    {
        HeadRow<T, VEC, LPH, AL> r;
        HeadRow<TG, VEC, LPH, AL> o;
        r.zero();
        o.zero();
        r.load(static_cast<const T*>(a.q) + L.it.x * a.q_row + L.head * a.q_head, L.j, a.dim);
        o.load(static_cast<const TG*>(a.dout) + L.it.x * a.do_row + L.head * a.do_head, L.j, a.dim);
        const float f = S::get(a.q_scale, L.it.x, a.heads, L.head) * a.scale * kLog2e;
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
        HeadRow<T, VEC, LPH, AL> kr[U], vr[U];
        float ks[U], vs[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            kr[u].zero();
            vr[u].zero();
            ks[u] = vs[u] = 1.0f;
            if (cur.ok[u]) {
                kr[u].load(k + cur.id[u] * a.k_row, L.j, a.dim);
                vr[u].load(v + cur.id[u] * a.v_row, L.j, a.dim);
                ks[u] = S::get(a.k_scale, cur.id[u], a.kv_heads, kvh);
                vs[u] = S::get(a.v_scale, cur.id[u], a.kv_heads, kvh);
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
        if (a.out) store_head<TG, VEC, LPH, AL>(static_cast<TG*>(a.out) + at * a.dim, L.j, a.dim, A);
        if (L.j == 0) a.stats[at] = make_float2(log2_total(m, l), delta);
    } else {
        float* part = a.parts + (static_cast<int64_t>(L.it.w) * a.heads + L.head) * (2 * a.dim + 3);
        if (L.j == 0) {
            part[0] = m;
            part[1] = l;
            part[2] = dsum;
        }
        store_part<VEC, LPH, AL>(part + 3, L.j, a.dim, A);
        store_part<VEC, LPH, AL>(part + 3 + a.dim, L.j, a.dim, B);
    }
}

template <typename T, typename TG, int VEC, int LPH, bool AL>
__global__ __launch_bounds__(256) void attn_bwd_kv_kernel(const AttnArgs a) {
    constexpr int U = kEdgesInFlight;
    typedef RowScale<T> S;
    const ItemLane L = item_lane<LPH>(a, a.kv_heads);
    if (!L.on) return;
    const T* q = static_cast<const T*>(a.q) + static_cast<int64_t>(L.head) * a.rep * a.q_head;
    const TG* o = static_cast<const TG*>(a.dout) + static_cast<int64_t>(L.head) * a.rep * a.do_head;
    float k[VEC], v[VEC], dk[VEC], dv[VEC];
    {
        HeadRow<T, VEC, LPH, AL> kr, vr;
        kr.zero();
        vr.zero();
        kr.load(static_cast<const T*>(a.k) + L.it.x * a.k_row + L.head * a.k_head, L.j, a.dim);
        vr.load(static_cast<const T*>(a.v) + L.it.x * a.v_row + L.head * a.v_head, L.j, a.dim);
        const float f = S::get(a.k_scale, L.it.x, a.kv_heads, L.head) * a.scale * kLog2e;
        const float fv = S::get(a.v_scale, L.it.x, a.kv_heads, L.head);
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
        if (e + U < end) next.load(a, e + U, end);
        for (int r = 0; r < a.rep; ++r) {
            HeadRow<T, VEC, LPH, AL> qr[U];
            HeadRow<TG, VEC, LPH, AL> gr[U];
            float qs[U];
            float2 st[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                qr[u].zero();
                gr[u].zero();
                qs[u] = 1.0f;
                st[u] = make_float2(0.0f, 0.0f);
                if (cur.ok[u]) {
                    const int h = L.head * a.rep + r;
                    qr[u].load(q + cur.id[u] * a.q_row + r * a.q_head, L.j, a.dim);
                    gr[u].load(o + cur.id[u] * a.do_row + r * a.do_head, L.j, a.dim);
                    qs[u] = S::get(a.q_scale, cur.id[u], a.heads, h);
                    st[u] = a.stats[static_cast<int64_t>(cur.id[u]) * a.heads + h];
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
                if constexpr (S::kScaled) t *= qs[u];
                const float p = cur.ok[u] ? exp2_fast(t - st[u].x) : 0.0f;
                float ds = cur.ok[u] ? p * (w - st[u].y) : 0.0f;
                if constexpr (S::kScaled) ds *= qs[u];
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
        if (a.out) store_head<TG, VEC, LPH, AL>(static_cast<TG*>(a.out) + at, L.j, a.dim, dk);
        if (a.out2) store_head<TG, VEC, LPH, AL>(static_cast<TG*>(a.out2) + at, L.j, a.dim, dv);
    } else {
        float* part = a.parts + (static_cast<int64_t>(L.it.w) * a.kv_heads + L.head) * (2 * a.dim);
        store_part<VEC, LPH, AL>(part, L.j, a.dim, dk);
        store_part<VEC, LPH, AL>(part + a.dim, L.j, a.dim, dv);
    }
}

// One workgroup per (row of several items, head): thread t holds element t % width, slice t / width of the parts.
struct JoinArgs {
    const int4* split;  // row, first part, last part + 1
    const float* parts;
    void *out, *out2;
    float2* stats;
    int heads, dim, width;  // width: the power of two that holds dim, at most 256
    float scale;
};

enum JoinKind { kJoinForward, kJoinQuery, kJoinKeyValue };

__device__ __forceinline__ float block_max(float v, float* red) {
    v = wave_max(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}

__device__ __forceinline__ float block_sum(float v, float* red) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

template <typename T, int KIND>
__global__ __launch_bounds__(256) void attn_join_kernel(const JoinArgs a) {
    __shared__ float red[4];
    __shared__ float one[256], two[256];
    const int4 sp = a.split[blockIdx.x / a.heads];
    const int head = blockIdx.x % a.heads;
    const int n = sp.z - sp.y;
    constexpr int kHead = KIND == kJoinForward ? 2 : KIND == kJoinQuery ? 3 : 0;
    const int64_t len = (KIND == kJoinForward ? 1 : 2) * a.dim + kHead;
    const int64_t step = len * a.heads;
    const float* p = a.parts + (static_cast<int64_t>(sp.y) * a.heads + head) * len;
    const int d = threadIdx.x & (a.width - 1), slice = threadIdx.x / a.width, slices = 256 / a.width;
    float m = -INFINITY, l = 0.0f, dsum = 0.0f;
    if constexpr (KIND != kJoinKeyValue) {
        for (int i = threadIdx.x; i < n; i += 256) m = fmaxf(m, p[i * step]);
        m = block_max(m, red);
        const float shift = shift_of(m);
        for (int i = threadIdx.x; i < n; i += 256) {
            const float c = exp2_fast(p[i * step] - shift);
            l += p[i * step + 1] * c;
            if constexpr (KIND == kJoinQuery) dsum += p[i * step + 2] * c;
        }
        l = block_sum(l, red);
        if constexpr (KIND == kJoinQuery) dsum = block_sum(dsum, red);
    }
    float x = 0.0f, y = 0.0f;
    if (d < a.dim) {
        const float shift = shift_of(m);
        for (int i = slice; i < n; i += slices) {
            const float* r = p + i * step;
            const float c = KIND == kJoinKeyValue ? 1.0f : exp2_fast(r[0] - shift);
            x = __builtin_fmaf(r[kHead + d], c, x);
            if constexpr (KIND != kJoinForward) y = __builtin_fmaf(r[kHead + a.dim + d], c, y);
        }
    }
    one[threadIdx.x] = x;
    if constexpr (KIND != kJoinForward) two[threadIdx.x] = y;
    __syncthreads();
    if (slice != 0 || d >= a.dim) return;
    for (int s = 1; s < slices; ++s) {
        x += one[s * a.width + d];
        if constexpr (KIND != kJoinForward) y += two[s * a.width + d];
    }
    const int64_t at = static_cast<int64_t>(sp.x) * a.heads + head;
    const float r = l == 0.0f ? 0.0f : 1.0f / l;
    if constexpr (KIND == kJoinForward) {
        static_cast<T*>(a.out)[at * a.dim + d] = static_cast<T>(x * r);
    } else if constexpr (KIND == kJoinQuery) {
        const float delta = dsum * r;
        if (a.out) static_cast<T*>(a.out)[at * a.dim + d] = static_cast<T>((x - delta * y) * (a.scale * r));
        if (d == 0) a.stats[at] = make_float2(log2_total(m, l), delta);
    } else {
        if (a.out) static_cast<T*>(a.out)[at * a.dim + d] = static_cast<T>(x * a.scale);
        if (a.out2) static_cast<T*>(a.out2)[at * a.dim + d] = static_cast<T>(y);
    }
}

enum AttnPass { kPassForward, kPassQuery, kPassKeyValue };

// Launches one pass over `items` and its join; `aligned`: rows are reached by vector loads.  T: fp32 / bf16 / fp16
// operands, or int8_t checkpoints under results of type TG.  False: a grid beyond the device's limit.
template <typename T, typename TG>
bool launch_attention(AttnPass pass, AttnArgs a, JoinArgs j, int64_t num_split, bool aligned, hipStream_t s);

template <typename T, typename TG, int VEC, int LPH, bool AL>
bool launch_attention_lanes(AttnPass pass, AttnArgs& a, hipStream_t s) {
    const int heads = pass == kPassKeyValue ? a.kv_heads : a.heads;
    // 128 bytes of a gathered row: eight lanes of 16 bytes, as far as there are heads
    a.tile_log = 0;
    while ((LPH << a.tile_log) < 8 && (1 << a.tile_log) < heads) ++a.tile_log;
    a.tiles = static_cast<int>(ceil_div(heads, 1 << a.tile_log));
    const int64_t per_block = 256 / (LPH << a.tile_log);
    const int64_t blocks = ceil_div(a.num_items, per_block) * a.tiles;
    if (blocks > 0x7fffffffLL) return false;
    if (blocks == 0) return true;
    const dim3 grid(static_cast<uint32_t>(blocks)), block(256);
    if (pass == kPassForward) {
        if constexpr (__is_same(T, TG)) hipLaunchKernelGGL((attn_fwd_kernel<T, VEC, LPH, AL>), grid, block, 0, s, a);
    } else if (pass == kPassQuery) {
        hipLaunchKernelGGL((attn_bwd_q_kernel<T, TG, VEC, LPH, AL>), grid, block, 0, s, a);
    } else {
        hipLaunchKernelGGL((attn_bwd_kv_kernel<T, TG, VEC, LPH, AL>), grid, block, 0, s, a);
    }
    return true;
}

template <typename T, typename TG, int VEC, bool AL>
bool launch_attention_vec(AttnPass pass, AttnArgs& a, hipStream_t s) {
    const int pieces = (a.dim + VEC - 1) / VEC;
    if (pieces <= 1) return launch_attention_lanes<T, TG, VEC, 1, AL>(pass, a, s);
    if (pieces <= 2) return launch_attention_lanes<T, TG, VEC, 2, AL>(pass, a, s);
    if (pieces <= 4) return launch_attention_lanes<T, TG, VEC, 4, AL>(pass, a, s);
    if (pieces <= 8) return launch_attention_lanes<T, TG, VEC, 8, AL>(pass, a, s);
    if (pieces <= 16) return launch_attention_lanes<T, TG, VEC, 16, AL>(pass, a, s);
    if (pieces <= 32) return launch_attention_lanes<T, TG, VEC, 32, AL>(pass, a, s);
    if constexpr (VEC == 4) return launch_attention_lanes<T, TG, VEC, 64, AL>(pass, a, s);
    return false;
}

template <typename T, typename TG>
bool launch_attention(AttnPass pass, AttnArgs a, JoinArgs j, int64_t num_split, bool aligned, hipStream_t s) {
    constexpr int VEC = sizeof(T) == 4 ? 4 : 8;
    const bool ok = aligned ? launch_attention_vec<T, TG, VEC, true>(pass, a, s) : launch_attention_vec<T, TG, VEC, false>(pass, a, s);
    if (!ok) return false;
    if (num_split == 0) return true;
    const int64_t blocks = num_split * j.heads;
    if (blocks > 0x7fffffffLL) return false;
    const dim3 grid(static_cast<uint32_t>(blocks)), block(256);
    if (pass == kPassForward)
        hipLaunchKernelGGL((attn_join_kernel<TG, kJoinForward>), grid, block, 0, s, j);
    else if (pass == kPassQuery)
        hipLaunchKernelGGL((attn_join_kernel<TG, kJoinQuery>), grid, block, 0, s, j);
    else
        hipLaunchKernelGGL((attn_join_kernel<TG, kJoinKeyValue>), grid, block, 0, s, j);
    return true;
}

}  // namespace tango
