// Weight and bias gradient of a linear layer whose input was kept as an 8-bit checkpoint:
//   dW[n, k] = sum over rows m of dy[m, n] x[m, k],  x[m, k] = q[m, k] s[m, run of k],      db[n] = sum over m of dy[m, n].
//
// On the matrix cores in bf16 without losing fp32's precision: the integers q are exact in bf16 (8 bits), and the scale,
// constant over a run, goes to the other factor: dW[n, k] = sum (dy[m, n] s[m]) q[m, k].  The product dy s, one fp32
// rounding, is split into bf16 terms (each the rounding of what the ones before left): three terms hold all 24 bits of
// an fp32 product, two (16 bits, an error of 2^-17 at most) are well below the rounding of a 16-bit result.  Sums are fp32.
//
// A workgroup owns a tile of kTileN x kTileK results inside one run and a share of the rows, kStep rows at a time: every
// thread loads eight rows of a column (so the transposition that the matrix instructions want costs nothing), scales,
// splits and writes 16 bytes of eight consecutive rows per term to LDS; four waves own a quarter of the tile each.
// The next step's loads are in flight while a step is multiplied.  LDS is laid out [row octet][column][8 rows]: both the
// writes and the fragment reads of neighbouring lanes are neighbouring 16-byte pieces.  Partial sums of the row shares
// go to a slab each and a second kernel adds the slabs in order.  The tiles of one row share are neighbours on one XCD,
// so dy and q come from HBM once and from that XCD's L2 for the other tiles.
#include "element.hpp"

namespace tango {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kTileN = 128, kTileK = 128, kStep = 32;

struct WGradArgs {
    const void* dy;
    const int8_t* q;
    const float* scale;
    float *slab, *slab_b;  // [splits, N, K], [splits, N]
    int64_t ldy, ldq, M, m_share;
    int N, K, group, runs, tiles_run, tiles_k, tiles, splits;
    int pairs, quads;  // dy in 2-element loads (16-bit types), q in 4-byte loads
};

// The column order inside a tile's LDS rows: what one thread loads together lies kTile / width apart, so that the
// writes of neighbouring threads are neighbours.
template <int WIDTH, int TILE>
__device__ __forceinline__ int column_of(int slot) {
    return (slot % (TILE / WIDTH)) * WIDTH + slot / (TILE / WIDTH);
}

__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
    const uint32_t lo = __builtin_bit_cast(uint16_t, static_cast<bf16_t>(a));
    const uint32_t hi = __builtin_bit_cast(uint16_t, static_cast<bf16_t>(b));
    return lo | (hi << 16);
}

template <typename T, int TERMS>
__global__ __launch_bounds__(256) void weight_grad_kernel(const WGradArgs a) {
    constexpr int W = sizeof(T) == 4 ? 1 : 2;               // columns of dy a thread loads together
    constexpr int ITEMS = kTileN / W * (kStep / 8) / 256;   // (columns, octet) pieces per thread
    __shared__ u32x4 lds_a[2][TERMS][kStep / 8][kTileN];
    __shared__ u32x4 lds_b[2][kStep / 8][kTileK];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
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
    const int k0 = run * a.group + (tk - run * a.tiles_run) * kTileK;
    const int k_end = k0 + kTileK < run_end ? k0 + kTileK : run_end;
    const int64_t m_begin = split * a.m_share;
    const int64_t m_end = m_begin + a.m_share < a.M ? m_begin + a.m_share : a.M;
    const bool want_b = a.slab_b && tk == 0;

    const T* dy = static_cast<const T*>(a.dy);
    Pack<T, W> ra[ITEMS][8];
    float rs[ITEMS][8];
    uint32_t rq[4];
    float bsum[ITEMS][W];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int w = 0; w < W; ++w) bsum[i][w] = 0.0f;

    // this thread's pieces: dy columns and octet, q columns and half octet
    int col[ITEMS], oct[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int id = tid + 256 * i;
        col[i] = id % (kTileN / W);
        oct[i] = id / (kTileN / W);
    }
    const int kc = tid % (kTileK / 4), mq = tid / (kTileK / 4);
    const int kq = k0 + 4 * kc;

    auto load = [&](int64_t m0) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int n = n0 + col[i] * W;
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                const int64_t m = m0 + oct[i] * 8 + r;
                const bool ok = m < m_end && n < a.N;
                ra[i][r].zero();
                rs[i][r] = 0.0f;
                if (ok) {
                    const T* p = dy + m * a.ldy + n;
                    if constexpr (W == 1) {
                        ra[i][r].load(p);
                    } else if (a.pairs && n + 1 < a.N) {
                        ra[i][r].load(p);
                    } else {
                        const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
                        ra[i][r].w[0] = h[0] | (n + 1 < a.N ? static_cast<uint32_t>(h[1]) << 16 : 0u);
                    }
                    rs[i][r] = a.scale[m * a.runs + run];
                }
            }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int64_t m = m0 + mq * 4 + r;
            rq[r] = 0;
            if (m < m_end && kq < k_end) {
                const int8_t* p = a.q + m * a.ldq + kq;
                if (a.quads && kq + 3 < a.K) {
                    rq[r] = *reinterpret_cast<const uint32_t*>(p);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (kq + j < k_end) rq[r] |= static_cast<uint32_t>(static_cast<uint8_t>(p[j])) << (8 * j);
                }
            }
        }
    };
    auto store = [&](int buf, int64_t m0) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int w = 0; w < W; ++w) {
                float x[8];
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    const float d = ra[i][r].get(w);
                    bsum[i][w] += d;
                    // rows past the end hold zeros, whatever their scale
                    x[r] = m0 + oct[i] * 8 + r < m_end ? d * rs[i][r] : 0.0f;
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
                    lds_a[buf][t][oct[i]][w * (kTileN / W) + col[i]] = o;
                }
            }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float x[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] = static_cast<float>(static_cast<int8_t>(rq[r] >> (8 * j)));
            u32x2 o;
            o[0] = bf16_pair(x[0], x[1]);
            o[1] = bf16_pair(x[2], x[3]);
            reinterpret_cast<u32x2*>(&lds_b[buf][mq >> 1][j * (kTileK / 4) + kc])[mq & 1] = o;
        }
    };

    f32x16 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
    const int wn = (wave >> 1) * 64 + (lane & 31), wk = (wave & 1) * 64 + (lane & 31), half = lane >> 5;

    if (m_begin < m_end) {
        load(m_begin);
        store(0, m_begin);
    }
    __syncthreads();
    int buf = 0;
    for (int64_t m0 = m_begin; m0 < m_end; m0 += kStep) {
        const bool more = m0 + kStep < m_end;
        if (more) load(m0 + kStep);
#pragma unroll
        for (int s = 0; s < kStep / 16; ++s) {
            bf16x8 fb[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) fb[j] = __builtin_bit_cast(bf16x8, lds_b[buf][2 * s + half][wk + 32 * j]);
#pragma unroll
            for (int t = 0; t < TERMS; ++t)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const bf16x8 fa = __builtin_bit_cast(bf16x8, lds_a[buf][t][2 * s + half][wn + 32 * i]);
#pragma unroll
                    for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa, fb[j], acc[i][j], 0, 0, 0);
                }
        }
        if (more) store(buf ^ 1, m0 + kStep);
        __syncthreads();
        buf ^= 1;
    }

    float* slab = a.slab + static_cast<int64_t>(split) * a.N * a.K;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int sn = (wave >> 1) * 64 + 32 * i + 8 * (r / 4) + 4 * half + (r & 3);
                const int n = n0 + column_of<W, kTileN>(sn);
                const int k = k0 + column_of<4, kTileK>(wk + 32 * j);
                if (n < a.N && k < k_end) slab[static_cast<int64_t>(n) * a.K + k] = acc[i][j][r];
            }
    if (want_b) {  // the octets' sums of a column, in octet order
        float* sums = reinterpret_cast<float*>(lds_a);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int w = 0; w < W; ++w) sums[oct[i] * kTileN + col[i] * W + w] = bsum[i][w];
        __syncthreads();
        if (tid < kTileN && n0 + tid < a.N) {
            float t = 0.0f;
            for (int o = 0; o < kStep / 8; ++o) t += sums[o * kTileN + tid];
            a.slab_b[static_cast<int64_t>(split) * a.N + n0 + tid] = t;
        }
    }
}

// Adds the row shares' slabs in order; the last workgroups do the bias.
template <typename T>
__global__ __launch_bounds__(256) void weight_grad_sum_kernel(T* dw, T* db, const float* slab, const float* slab_b, int64_t count,
                                                              int n, int splits) {
    const int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const bool bias = id >= count;
    const float* p = bias ? slab_b : slab;
    const int64_t at = bias ? id - count : id, step = bias ? n : count;
    if (bias && (!db || at >= n)) return;
    float t = 0.0f;
    int s = 0;
    for (; s + 4 <= splits; s += 4) {
        const float x0 = p[s * step + at], x1 = p[(s + 1) * step + at], x2 = p[(s + 2) * step + at], x3 = p[(s + 3) * step + at];
        t = (((t + x0) + x1) + x2) + x3;
    }
    for (; s < splits; ++s) t += p[s * step + at];
    (bias ? db : dw)[at] = static_cast<T>(t);
}

struct WGradPlan {
    int64_t runs, tiles_run, tiles_k, tiles, splits, m_share, slab_floats;
};

static WGradPlan wgrad_plan(int64_t M, int64_t N, int64_t K, int64_t group) {
    WGradPlan p;
    if (group > K) group = K;
    p.runs = ceil_div(K, group);
    p.tiles_run = ceil_div(group, kTileK);
    const int64_t last = K - (p.runs - 1) * group;
    p.tiles_k = (p.runs - 1) * p.tiles_run + ceil_div(last, kTileK);
    p.tiles = p.tiles_k * ceil_div(N, kTileN);
    // two workgroups for each CU, each at least four steps of rows
    int64_t splits = ceil_div(512, p.tiles);
    const int64_t most = ceil_div(M, 4 * kStep);
    if (splits > most) splits = most;
    if (splits < 1) splits = 1;
    p.m_share = ceil_div(ceil_div(M, splits), kStep) * kStep;
    p.splits = p.m_share ? ceil_div(M, p.m_share) : 1;
    p.slab_floats = p.splits * N * (K + 1);
    return p;
}

template <typename T, int TERMS>
static void launch_weight_grad(const WGradArgs& a, void* dw, void* db, hipStream_t s) {
    const int64_t blocks = static_cast<int64_t>(a.splits >= 8 ? (a.splits + 7) / 8 * 8 : a.splits) * a.tiles;
    hipLaunchKernelGGL((weight_grad_kernel<T, TERMS>), dim3(static_cast<uint32_t>(blocks)), dim3(256), 0, s, a);
    const int64_t count = static_cast<int64_t>(a.N) * a.K;
    hipLaunchKernelGGL((weight_grad_sum_kernel<T>), dim3(static_cast<uint32_t>(ceil_div(count + (db ? a.N : 0), 256))), dim3(256), 0, s,
                       static_cast<T*>(dw), static_cast<T*>(db), a.slab, a.slab_b, count, a.N, a.splits);
}

// sizes whose tile counts and offsets into a slab stay within the kernels' 32-bit numbers
static bool wgrad_sizes(int64_t M, int64_t N, int64_t K) {
    return M < (1LL << 31) && N <= 65536 && K <= 65536;
}

}  // namespace tango

using namespace tango;

extern "C" {

size_t tango_weight_grad_i8_workspace(int64_t M, int64_t N, int64_t K, int64_t group) {
    if (M <= 0 || N <= 0 || K <= 0 || group <= 0 || !wgrad_sizes(M, N, K)) return 0;
    return static_cast<size_t>(wgrad_plan(M, N, K, group).slab_floats) * 4;
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
    const WGradPlan p = wgrad_plan(M, N, K, group);
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
    a.tiles_run = static_cast<int>(p.tiles_run);
    a.tiles_k = static_cast<int>(p.tiles_k);
    a.tiles = static_cast<int>(p.tiles);
    a.splits = static_cast<int>(p.splits);
    a.pairs = ldy % 2 == 0 && aligned_to(dy, 4);
    a.quads = ldq % 4 == 0 && aligned_to(q, 4) && (p.runs == 1 || group % 4 == 0);
    if (dtype == TANGO_F32)
        launch_weight_grad<float, 3>(a, dw, db, as_stream(stream));
    else if (dtype == TANGO_BF16)
        launch_weight_grad<bf16_t, 2>(a, dw, db, as_stream(stream));
    else
        launch_weight_grad<f16_t, 2>(a, dw, db, as_stream(stream));
    return launch_status();
}

}  // extern "C"
