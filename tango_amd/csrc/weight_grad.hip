// Weight and bias gradient of a linear layer whose input was kept as an 8-bit checkpoint:
//   dW[n, k] = sum over rows m of dy[m, n] x[m, k],  x[m, k] = q[m, k] s[m, run of k],      db[n] = sum over m of dy[m, n].
//
// On the matrix cores in bf16 without losing fp32's precision: the integers q are exact in bf16 (8 bits), and the scale,
// constant over a run, goes to the other factor: dW[n, k] = sum (dy[m, n] s[m]) q[m, k].  The product dy s, one fp32
// rounding, is split into bf16 terms (each the rounding of what the ones before left): three terms hold all 24 bits of
// an fp32 product, two (16 bits, an error of 2^-17 at most) are well below the rounding of a 16-bit result.  Sums are fp32.
//
// A workgroup owns a tile of kTileN x at most kTileK results inside one run and a share of the rows, kStep rows at a
// time.  Each of its four waves loads eight rows (so their scales are scalar), a lane two columns of dy and four of q;
// a thread holds eight rows of a column, so the transposition that the matrix instructions want costs nothing, and
// writes 16 bytes of eight consecutive rows per column and term to LDS.  Then each wave multiplies 32 of the tile's
// dy columns with all of its q columns: 32x32x16, accumulators in registers.  The next step's loads are in flight while
// a step is multiplied, and two workgroups a CU overlap one's conversions with the other's matrix instructions.
// LDS is laid out [row octet][column][8 rows]: writes and fragment reads of neighbouring lanes are neighbouring 16-byte
// pieces.  Partial sums of the row shares go to a slab each and a second kernel adds the slabs in order.  The tiles of
// one row share are neighbours on one XCD, so dy and q come from HBM once and from that XCD's L2 for the other tiles.
//
// Measured, [232965, 256] x [232965, 602] fp32 (three tiles of 224 columns): 269 us and 11 us for the slabs; the matrix
// instructions alone are 229 k cycles a SIMD of the 502 k at 1.9 GHz.  On the way: 128 x 128 tiles with the conversions
// between the matrix instructions' steps 785 us; scalar loads of the scales (they share the counter of LDS reads) and a
// branch per 32 columns 457 us; one workgroup a CU for want of LDS, or 66 workgroups on some XCDs' 64 places, 336 us.
// A plain large product runs at 1.2 PFLOP/s here: three terms take 200 us at that rate.
#include <math.h>

#include "element.hpp"

namespace tango {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kTileN = 128, kTileK = 256, kStep = 32, kSub = 32;

struct WGradArgs {
    const void* dy;
    const int8_t* q;
    const float* scale;
    float *slab, *slab_b;  // [splits, N, K], [splits, N]
    int64_t ldy, ldq, M, m_share;
    int N, K, group, runs, tile_k, tiles_run, tiles_k, tiles, splits;
};

__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const f32x2 v = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
}

// Columns and slots.  Slot 64 w + l of a dy row holds column 2 l + w (a lane writes its columns 2 l and 2 l + 1 beside its
// neighbours'); the smallest column of the 32 slots from s on is that of s.
__device__ __forceinline__ int n_column(int slot) { return 2 * (slot & 63) + (slot >> 6); }
// Column 4 l + j of a q row, in a piece of 8 SUBS slots for each j.  A fragment of 32 neighbouring columns reads eight
// slots (128 bytes) of each piece; pieces read together lie in different banks (256 bytes) if an odd piece starts on an
// odd multiple of 128 bytes: for an odd SUBS it does, else it is turned by eight slots.
template <int SUBS>
__device__ __forceinline__ int k_slot(int j, int l) {
    if constexpr (SUBS % 2 == 0) l = l + 8 * (j & 1) < 8 * SUBS ? l + 8 * (j & 1) : l + 8 - 8 * SUBS;
    return j * (8 * SUBS) + l;
}
__device__ __forceinline__ int k_column(int sub, int col) { return kSub * sub + 4 * (col & 7) + (col >> 3); }

// A wave's eight rows of one step in registers.
template <typename T>
struct WGradStage {
    Pack<T, 2> dy[8];
    uint32_t q[8];
    float scale;  // lane l: that of row l % 8
};

// A load whose base is the same in all lanes and stays in scalar registers, plus a 32-bit offset per lane (left alone, the
// compiler adds the lane's offset first and holds sixteen 64-bit addresses in vector registers).
template <typename V, typename P>
__device__ __forceinline__ V load_from(const P* base, uint32_t offset) {
    typedef const V __attribute__((address_space(1), aligned(1))) * Global;
    uint64_t at = reinterpret_cast<uint64_t>(base);
    asm("" : "+s"(at));
    return *reinterpret_cast<Global>(at + offset);
}

// One for a row that is there, zero for one that is not: a scalar, which the compiler is not to turn into a selection in
// every lane.
__device__ __forceinline__ float presence(bool there) {
    uint32_t b = there ? 0x3f800000u : 0u;
    asm("" : "+s"(b));
    return __uint_as_float(b);
}

// WHOLE: dy in loads of two columns (N > 1), q in loads of four (runs and rows of q start on multiples of four), both
// unconditional: columns past the end are moved back inside, what they give is not used.  Otherwise an element at a time.
template <typename T, int TERMS, int SUBS, bool WHOLE>
__global__ __launch_bounds__(256, 2) void weight_grad_kernel(const WGradArgs a) {
    // [buffer][term, then q][octet][column]
    constexpr int kA = TERMS * (kStep / 8) * kTileN, kB = (kStep / 8) * SUBS * kSub;
    extern __shared__ u32x4 lds[];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int split, tile;
    if (a.splits >= 8) {  // a split's tiles stay on one XCD
        const int j = blockIdx.x >> 3;
        split = (blockIdx.x & 7) + 8 * (j / a.tiles);
        tile = j % a.tiles;
        if (split >= a.splits) return;
    } else {
        split = blockIdx.x / a.tiles;
        tile = blockIdx.x % a.tiles;
    }
    const int tk = tile % a.tiles_k, n0 = tile / a.tiles_k * kTileN;
    const int run = tk / a.tiles_run;
    const int run_end = run == a.runs - 1 ? a.K : (run + 1) * a.group;
    const int k0 = run * a.group + (tk - run * a.tiles_run) * a.tile_k;
    const int k_end = k0 + a.tile_k < run_end ? k0 + a.tile_k : run_end;
    const int64_t m_begin = split * a.m_share;
    const int64_t m_end = m_begin + a.m_share < a.M ? m_begin + a.m_share : a.M;
    const bool want_b = a.slab_b && tk == 0;

    // This lane's columns.  If N is odd, the lane of the last column loads the pair that ends with it, one column early.
    const int n = n0 + 2 * lane, k = k0 + 4 * lane;
    const int n_at = n + 1 < a.N ? n : a.N - 2, k_at = k < k_end ? k : k0;

    float bsum[2] = {0.0f, 0.0f};

    // the wave's eight rows from `first` on; rows past `last` are that row again, and convert drops them
    auto load_rows = [&](WGradStage<T>& st, int64_t first, int last) {
        const T* dy = static_cast<const T*>(a.dy) + first * a.ldy;
        const int8_t* q = a.q + first * a.ldq;
        if constexpr (WHOLE) {
            const uint32_t dy_at = static_cast<uint32_t>(n_at) * sizeof(T), q_at = static_cast<uint32_t>(k_at);
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                const int row = r < last ? r : last;
                if constexpr (sizeof(T) == 4) {
                    const u32x2 t = load_from<u32x2>(dy + row * a.ldy, dy_at);
                    st.dy[r].w[0] = t[0];
                    st.dy[r].w[1] = t[1];
                } else {
                    st.dy[r].w[0] = load_from<uint32_t>(dy + row * a.ldy, dy_at);
                }
                st.q[r] = load_from<uint32_t>(q + row * a.ldq, q_at);
            }
        } else {
            for (int r = 0; r < 8; ++r) {
                const int row = r < last ? r : last;
                Pack<T, 1> x, y;
                x.zero();
                y.zero();
                if (n < a.N) x.load(dy + row * a.ldy + n);
                if (n + 1 < a.N) y.load(dy + row * a.ldy + n + 1);
                uint32_t w = 0;
                for (int j = 0; j < 4; ++j)
                    if (k + j < k_end) w |= static_cast<uint32_t>(static_cast<uint8_t>(q[row * a.ldq + k + j])) << (8 * j);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i == r) {
                        if constexpr (sizeof(T) == 4) {
                            st.dy[i].w[0] = x.w[0];
                            st.dy[i].w[1] = y.w[0];
                        } else {
                            st.dy[i].w[0] = x.w[0] | (y.w[0] << 16);
                        }
                        st.q[i] = w;
                    }
            }
        }
        // one vector load: scalar loads share a counter with the LDS reads that the matrix instructions wait for
        const int sr = (lane & 7) < last ? (lane & 7) : last;
        st.scale = a.scale[(first + sr) * a.runs + run];
    };
    const int share = static_cast<int>(m_end - m_begin);
    auto rows_of = [&](int step) {  // of this wave: 0 .. 8
        const int left = share - step * kStep - wave * 8;
        return left >= 8 ? 8 : left > 0 ? left : 0;
    };
    auto load = [&](WGradStage<T>& st, int step) {
        const int64_t first = m_begin + static_cast<int64_t>(step) * kStep + wave * 8;
        const int rows = rows_of(step);
        if (rows == 8)
            load_rows(st, first, 7);
        else
            load_rows(st, rows > 0 ? first : m_end - 1, rows > 0 ? rows - 1 : 0);
    };
    // Rows that are not there repeat one that is, with a scale of zero: they add nothing to a finite sum (and one that is
    // not finite already holds that row).
    auto convert_dy = [&](const WGradStage<T>& st, u32x4* at, int rows) {
        float scale[8];
#pragma unroll
        for (int r = 0; r < 8; ++r)
            scale[r] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(st.scale), r) & (r < rows ? -1 : 0));
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            float x[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                bsum[w] = __builtin_fmaf(st.dy[r].get(w), presence(r < rows), bsum[w]);
                x[r] = st.dy[r].get(w) * scale[r];
            }
#pragma unroll
            for (int t = 0; t < TERMS; ++t) {
                u32x4 o;
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    o[p] = bf16_pair(x[2 * p], x[2 * p + 1]);
                    x[2 * p] -= __uint_as_float(o[p] << 16);
                    x[2 * p + 1] -= __uint_as_float(o[p] & 0xffff0000u);
                }
                at[(t * (kStep / 8) + wave) * kTileN + w * 64 + lane] = o;
            }
        }
    };
    const int k_lane = lane < 8 * SUBS ? lane : 0;
    auto convert_q = [&](const WGradStage<T>& st, u32x4* at) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float x[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) x[r] = static_cast<float>(static_cast<int8_t>(st.q[r] >> (8 * j)));
            u32x4 o;
#pragma unroll
            for (int p = 0; p < 4; ++p) o[p] = bf16_pair(x[2 * p], x[2 * p + 1]);
            // lanes without a column write what nothing reads
            u32x4* const to = at + kA + wave * (SUBS * kSub) + k_slot<SUBS>(j, k_lane);
            *(lane < 8 * SUBS ? to : lds + 2 * (kA + kB) + (lane & 7)) = o;
        }
    };

    f32x16 acc[SUBS];
#pragma unroll
    for (int j = 0; j < SUBS; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[j][r] = 0.0f;
    const int half = lane >> 5, col = lane & 31;
    auto multiply = [&](const u32x4* at, int s) {
        bf16x8 fa[TERMS], fb[SUBS];
#pragma unroll
        for (int t = 0; t < TERMS; ++t)
            fa[t] = __builtin_bit_cast(bf16x8, at[(t * (kStep / 8) + 2 * s + half) * kTileN + wave * 32 + col]);
#pragma unroll
        for (int j = 0; j < SUBS; ++j)
            fb[j] = __builtin_bit_cast(bf16x8, at[kA + (2 * s + half) * (SUBS * kSub) + k_slot<SUBS>(col >> 3, 8 * j + (col & 7))]);
#pragma unroll
        for (int t = 0; t < TERMS; ++t)
#pragma unroll
            for (int j = 0; j < SUBS; ++j) acc[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[t], fb[j], acc[j], 0, 0, 0);
    };
    // Order of issue inside a half step: the fragment reads, then a few vector instructions behind each matrix instruction.
    auto interleave = [&]() {
        __builtin_amdgcn_sched_group_barrier(0x100, TERMS + SUBS, 0);
#pragma unroll
        for (int m = 0; m < TERMS * SUBS; ++m) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, 7, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    };

    // While step i is multiplied, step i + 1 is converted into the other buffer (in the same stretch of code: vector and
    // matrix instructions of a wave overlap) and the loads of step i + 2 are on their way.  Steps in pairs: an odd
    // number is followed by one without rows.
    const int steps = (share + kStep - 1) / kStep;
    u32x4 *const buf0 = lds, *const buf1 = lds + kA + kB;
    WGradStage<T> s0, s1;
    auto step = [&](WGradStage<T>& loading, const WGradStage<T>& loaded, const u32x4* now, u32x4* next, int i) {
        load(loading, i + 2);
        const int rows = rows_of(i + 1);
        __builtin_amdgcn_sched_barrier(0);
        multiply(now, 0);
        convert_dy(loaded, next, rows);
        interleave();
        multiply(now, 1);
        convert_q(loaded, next);
        interleave();
        __syncthreads();
    };
    load(s0, 0);
    load(s1, 1);
    convert_dy(s0, buf0, rows_of(0));
    convert_q(s0, buf0);
    __syncthreads();
    for (int i = 0; i < steps; i += 2) {
        step(s0, s1, buf0, buf1, i);
        step(s1, s0, buf1, buf0, i + 1);
    }

    // what slot s holds: with an odd N the last lane's two slots hold the columns before and at the end
    auto result_column = [&](int s) {
        const int c = n0 + n_column(s);
        return WHOLE && (a.N & 1) && (c | 1) == a.N ? c - 1 : c;
    };
    float* slab = a.slab + static_cast<int64_t>(split) * a.N * a.K;
#pragma unroll
    for (int j = 0; j < SUBS; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int nn = result_column(wave * 32 + 8 * (r / 4) + 4 * half + (r & 3));
            const int kk = k0 + k_column(j, col);
            if (nn < a.N && kk < k_end) slab[static_cast<int64_t>(nn) * a.K + kk] = acc[j][r];
        }
    if (want_b) {  // the octets' sums of a column, in octet order
        float* sums = reinterpret_cast<float*>(lds);
        const bool early = WHOLE && n == a.N - 1;
        sums[wave * kTileN + 2 * lane] = early ? bsum[1] : bsum[0];
        sums[wave * kTileN + 2 * lane + 1] = bsum[1];
        __syncthreads();
        if (tid < kTileN && n0 + tid < a.N) {
            float t = 0.0f;
            for (int o = 0; o < kStep / 8; ++o) t += sums[o * kTileN + tid];
            a.slab_b[static_cast<int64_t>(split) * a.N + n0 + tid] = t;
        }
    }
}

// Adds the row shares' slabs: a workgroup owns 32 results, its eight groups of 32 lanes take every eighth slab, their sums
// are added in order (one lane for all slabs of a result: 50 us of the 65 for 482 slabs of [40, 128]).  Results past the
// weight's are the bias's.
template <typename T>
__global__ __launch_bounds__(256) void weight_grad_sum_kernel(T* dw, T* db, const float* slab, const float* slab_b, int64_t count,
                                                              int n, int splits) {
    __shared__ float part[8][32];
    const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
    const int64_t id = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    const bool bias = id >= count, on = id < count + (db ? n : 0);
    const float* p = bias ? slab_b + (id - count) : slab + id;
    const int64_t step = bias ? n : count;
    float t = 0.0f;
    if (on) {
#pragma unroll 4
        for (int s = slice; s < splits; s += 8) t += p[s * step];
    }
    part[slice][lane] = t;
    __syncthreads();
    if (slice || !on) return;
    for (int s = 1; s < 8; ++s) t += part[s][lane];
    if (bias)
        db[id - count] = static_cast<T>(t);
    else
        dw[id] = static_cast<T>(t);
}

struct WGradPlan {
    int64_t runs, tile_k, tiles_run, tiles_k, tiles, splits, m_share, slab_floats;
};

// Columns of q in a tile at most: two workgroups have to fit a CU's 160 KB of LDS, which they do at 76 KB each and did not at
// 80 KB (three terms, 256 columns).
static constexpr int most_columns(int terms) { return terms == 3 ? kTileK - kSub : kTileK; }
static int terms_of(int dtype) { return dtype == TANGO_F32 ? 3 : 2; }

static WGradPlan wgrad_plan(int dtype, int64_t M, int64_t N, int64_t K, int64_t group) {
    WGradPlan p;
    const int64_t widest = most_columns(terms_of(dtype));
    if (group > K) group = K;
    p.runs = ceil_div(K, group);
    // a run in equal tiles
    p.tile_k = ceil_div(ceil_div(group, ceil_div(group, widest)), kSub) * kSub;
    p.tiles_run = ceil_div(group, p.tile_k);
    const int64_t last = K - (p.runs - 1) * group;
    p.tiles_k = (p.runs - 1) * p.tiles_run + ceil_div(last, p.tile_k);
    p.tiles = p.tiles_k * ceil_div(N, kTileN);
    // as many as are resident together (two workgroups on each of an XCD's 32 CUs), no second round; each at least four
    // steps of rows
    int64_t splits = p.tiles <= 64 ? 8 * (64 / p.tiles) : 512 / p.tiles;
    const int64_t most = ceil_div(M, 4 * kStep);
    if (splits > most) splits = most;
    // a share more costs its slab written and read (some 4 TB/s), a share less its rows for the others (some 1.3 us a
    // step): the sum is smallest at their ratio's root (19717 rows, 256 x 500 fp32: 52 shares 37 us, 64 45 us, 26 51 us)
    const int64_t best = static_cast<int64_t>(sqrt(20000.0 * static_cast<double>(M) / (static_cast<double>(N) * static_cast<double>(K))));
    if (splits > best) splits = best;
    if (splits < 1) splits = 1;
    p.m_share = ceil_div(ceil_div(M, splits), kStep) * kStep;
    p.splits = p.m_share ? ceil_div(M, p.m_share) : 1;
    p.slab_floats = p.splits * N * (K + 1);
    return p;
}

template <typename T, int TERMS, int SUBS, bool WHOLE>
static bool launch_weight_grad_tile(const WGradArgs& a, hipStream_t s) {
    constexpr int kLds = 2 * (kStep / 8) * (TERMS * kTileN + SUBS * kSub) * 16 + (SUBS * kSub < 256 ? 128 : 0);
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(weight_grad_kernel<T, TERMS, SUBS, WHOLE>),
                            hipFuncAttributeMaxDynamicSharedMemorySize, kLds) != hipSuccess) {
        (void)hipGetLastError();
        return false;
    }
    const int64_t blocks = static_cast<int64_t>(a.splits >= 8 ? (a.splits + 7) / 8 * 8 : a.splits) * a.tiles;
    hipLaunchKernelGGL((weight_grad_kernel<T, TERMS, SUBS, WHOLE>), dim3(static_cast<uint32_t>(blocks)), dim3(256), kLds, s, a);
    return true;
}

template <typename T, int TERMS>
static bool launch_weight_grad(const WGradArgs& a, bool whole, void* dw, void* db, hipStream_t s) {
    bool ok = false;
    if (!whole) {
        ok = launch_weight_grad_tile<T, TERMS, most_columns(TERMS) / kSub, false>(a, s);
    } else {
        switch (a.tile_k / kSub) {
            case 1: ok = launch_weight_grad_tile<T, TERMS, 1, true>(a, s); break;
            case 2: ok = launch_weight_grad_tile<T, TERMS, 2, true>(a, s); break;
            case 3: ok = launch_weight_grad_tile<T, TERMS, 3, true>(a, s); break;
            case 4: ok = launch_weight_grad_tile<T, TERMS, 4, true>(a, s); break;
            case 5: ok = launch_weight_grad_tile<T, TERMS, 5, true>(a, s); break;
            case 6: ok = launch_weight_grad_tile<T, TERMS, 6, true>(a, s); break;
            case 7: ok = launch_weight_grad_tile<T, TERMS, 7, true>(a, s); break;
            case 8:
                if constexpr (TERMS == 2) ok = launch_weight_grad_tile<T, TERMS, 8, true>(a, s);
                break;
        }
    }
    if (!ok) return false;
    const int64_t count = static_cast<int64_t>(a.N) * a.K;
    hipLaunchKernelGGL((weight_grad_sum_kernel<T>), dim3(static_cast<uint32_t>(ceil_div(count + (db ? a.N : 0), 32))), dim3(256), 0, s,
                       static_cast<T*>(dw), static_cast<T*>(db), a.slab, a.slab_b, count, a.N, a.splits);
    return true;
}

// sizes whose tile counts and offsets into a slab stay within the kernels' 32-bit numbers
static bool wgrad_sizes(int64_t M, int64_t N, int64_t K) {
    return M <= (1LL << 30) && N <= 65536 && K <= 65536;
}

}  // namespace tango

using namespace tango;

extern "C" {

size_t tango_weight_grad_i8_workspace(int dtype, int64_t M, int64_t N, int64_t K, int64_t group) {
    if (!float_type(dtype) || M <= 0 || N <= 0 || K <= 0 || group <= 0 || !wgrad_sizes(M, N, K)) return 0;
    return static_cast<size_t>(wgrad_plan(dtype, M, N, K, group).slab_floats) * 4;
}

int tango_weight_grad_i8(void* dw, void* db, const void* dy, int dtype, int64_t ldy, const int8_t* q, int64_t ldq, const float* scale,
                         int64_t group, int64_t M, int64_t N, int64_t K, void* workspace, size_t workspace_bytes,
                         tango_stream_t stream) {
    if (!float_type(dtype)) return TANGO_ERR_UNSUPPORTED;
    if (M <= 0 || N < 0 || K < 0 || group <= 0 || ldy < 0 || ldq < 0) return TANGO_ERR_INVALID_ARG;
    if (N == 0 || K == 0) return TANGO_OK;
    if (!dw || !dy || !q || !scale || !aligned_to(dy, element_size(dtype)) || !aligned_to(dw, element_size(dtype)) ||
        !aligned_to(db, element_size(dtype)) || !aligned_to(scale, 4))
        return TANGO_ERR_INVALID_ARG;
    if (!wgrad_sizes(M, N, K)) return TANGO_ERR_UNSUPPORTED;
    const WGradPlan p = wgrad_plan(dtype, M, N, K, group);
    if (!workspace || workspace_bytes < static_cast<size_t>(p.slab_floats) * 4 || !aligned_to(workspace, 16)) return TANGO_ERR_WORKSPACE;
    if (p.tiles * (p.splits + 8) > 0x7fffffffLL) return TANGO_ERR_UNSUPPORTED;
    WGradArgs a;
    a.dy = dy;
    a.q = q;
    a.scale = scale;
    a.slab = static_cast<float*>(workspace);
    a.slab_b = db ? a.slab + p.splits * N * K : nullptr;
    a.ldy = ldy;
    a.ldq = ldq;
    a.M = M;
    a.m_share = p.m_share;
    a.N = static_cast<int>(N);
    a.K = static_cast<int>(K);
    a.group = static_cast<int>(group > K ? K : group);
    a.runs = static_cast<int>(p.runs);
    a.tile_k = static_cast<int>(p.tile_k);
    a.tiles_run = static_cast<int>(p.tiles_run);
    a.tiles_k = static_cast<int>(p.tiles_k);
    a.tiles = static_cast<int>(p.tiles);
    a.splits = static_cast<int>(p.splits);
    const bool whole = N > 1 && ldq % 4 == 0 && ldq >= ceil_div(K, 4) * 4 && aligned_to(q, 4) && (p.runs == 1 || group % 4 == 0);
    const bool ok = dtype == TANGO_F32    ? launch_weight_grad<float, 3>(a, whole, dw, db, as_stream(stream))
                    : dtype == TANGO_BF16 ? launch_weight_grad<bf16_t, 2>(a, whole, dw, db, as_stream(stream))
                                          : launch_weight_grad<f16_t, 2>(a, whole, dw, db, as_stream(stream));
    return ok ? launch_status() : TANGO_ERR_LAUNCH;
}

}  // extern "C"
