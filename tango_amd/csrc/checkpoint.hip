// 8-bit checkpoints of activations: a row-major [rows, cols] tensor as int8 with one fp32 scale per run of `group`
// consecutive columns of a row (the last run of a row may be shorter), and back.
//
//   s = max|x| / 127 over the run (fp32),   q = the integer nearest to 127 x / max|x|, ties to even,   value q s.
//
// The quotient is decided exactly, not on a rounded 1/s: max|x| is a value of the run, so quotients that are ties
// (x = max|x| / 2 gives 63.5) are common in 16-bit data, and an approximate reciprocal would round them either way.
// A run that holds an infinity or a NaN cannot be held in 8 bits: its scale is NaN and its integers are 0, so every
// value of it comes back as NaN.  A run of zeros has scale 0.
//
// Both directions are bound by HBM: 4 or 2 bytes per element one way, 1 byte plus 4 / group the other.  A run is held
// in registers between its maximum and its rounding, so each element is read once.
#include "element.hpp"

namespace tango {

struct PackArgs {
    const void* x;
    int8_t* q;
    float* scale;
    int64_t rows, ldx, ldq, scale_row, scale_run;
    uint32_t total;  // runs of this launch: rows * groups
    int cols, group, lanes;  // lanes: a power of two, one run each lane group
    FastDiv groups;
};

// The nearest integer to 127 |x| / top.  xs = |x| and ts = top, both scaled by the power of two that brings top into
// [0.5, 1); inv ~ 127 / ts.  k = floor of the approximate quotient is off by at most one, and whichever side it fell
// on, the quotient lies in [k, k + 1] up to rounding errors far below a half: it rounds up exactly if it exceeds
// h = k + 1/2.  127 xs - h ts is compared with zero through the two halves of h ts (p + e, e from one fma): the fma
// 127 xs - p is exact whenever it is of e's size.
__device__ __forceinline__ int nearest_127(float xs, float ts, float inv) {
    const float k = floorf(xs * inv);
    const float h = k + 0.5f;
    const float p = h * ts;
    const float e = __builtin_fmaf(h, ts, -p);
    const float d = __builtin_fmaf(127.0f, xs, -p);
    const int n = static_cast<int>(k);
    return n + ((d > e || (d == e && (n & 1))) ? 1 : 0);
}

// The largest scale whose 127-fold is finite in fp32: fp32's largest number / 127, rounded down.  The nearest scale of
// a run that reaches that number would bring it back as an infinity.
constexpr float kLargestScale = 0x1.0204060000000p+121f;

struct RunScale {
    float top, inv;  // scaled to [0.5, 1); 127 / top
    int exp;
    float scale;
};

__device__ __forceinline__ RunScale run_scale(uint32_t top_bits) {
    RunScale r;
    const float top = __uint_as_float(top_bits);
    if (top_bits >= 0x7f800000u) {
        r.top = 1.0f;
        r.inv = 0.0f;  // unused: the integers of such a run are 0
        r.exp = 0;
        r.scale = __uint_as_float(0x7fc00000u);
    } else if (top_bits == 0) {
        r.top = 1.0f;
        r.inv = 127.0f;
        r.exp = 0;
        r.scale = 0.0f;
    } else {
        r.exp = __builtin_amdgcn_frexp_expf(top);
        r.top = __builtin_amdgcn_ldexpf(top, -r.exp);
        r.inv = 127.0f / r.top;
        r.scale = fminf(top / 127.0f, kLargestScale);
    }
    return r;
}

__device__ __forceinline__ int run_quant(float x, const RunScale& r) {
    const int n = nearest_127(__builtin_amdgcn_ldexpf(fabsf(x), -r.exp), r.top, r.inv);
    return x < 0.0f ? -n : n;
}

// Maximum over `lanes` (a power of two) neighbouring lanes, in all of them.  Non-negative floats as their bits: a NaN
// is the largest.
__device__ __forceinline__ uint32_t lanes_umax(uint32_t v, int lanes) {
    for (int off = 1; off < lanes; off <<= 1) {
        const uint32_t o = __shfl_xor(v, off, kWave);
        v = o > v ? o : v;
    }
    return v;
}

// `lanes` lanes own a run, R pieces of VEC elements each; UN runs per lane group are in flight together.
template <typename T, int VEC, int R, int UN>
__global__ __launch_bounds__(256) void pack_kernel(const PackArgs a) {
    const int lane = threadIdx.x & (a.lanes - 1);
    const uint32_t per_block = 256 / a.lanes;
    const uint32_t stride = gridDim.x * per_block;
    for (uint32_t first = blockIdx.x * per_block + threadIdx.x / a.lanes; first < a.total; first += stride * UN) {
        Pack<T, VEC> in[UN][R];
        uint32_t top[UN];
        int64_t row[UN];
        int col[UN], len[UN];
        uint32_t run[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const uint32_t id = first + u * stride;
            const bool ok = id < a.total;
            const uint32_t rw = a.groups.div(ok ? id : 0);
            row[u] = rw;
            run[u] = (ok ? id : 0) - rw * a.groups.d;
            col[u] = static_cast<int>(run[u]) * a.group;
            len[u] = ok ? (a.cols - col[u] < a.group ? a.cols - col[u] : a.group) : 0;
            const T* src = static_cast<const T*>(a.x) + row[u] * a.ldx + col[u];
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const int c = (i * a.lanes + lane) * VEC;
                in[u][i].zero();
                if (c < len[u]) in[u][i].load(src + c);
            }
        }
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            uint32_t t = 0;
#pragma unroll
            for (int i = 0; i < R; ++i)
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const uint32_t b = __float_as_uint(in[u][i].get(j)) & 0x7fffffffu;
                    t = b > t ? b : t;
                }
            top[u] = lanes_umax(t, a.lanes);
        }
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            if (!len[u]) continue;
            const RunScale r = run_scale(top[u]);
            int8_t* dst = a.q + row[u] * a.ldq + col[u];
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const int c = (i * a.lanes + lane) * VEC;
                if (c >= len[u]) continue;
                Pack<int8_t, VEC> o;
                o.zero();
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const int n = top[u] >= 0x7f800000u ? 0 : run_quant(in[u][i].get(j), r);
                    o.w[j / 4] |= (static_cast<uint32_t>(n) & 0xffu) << (8 * (j & 3));
                }
                o.store(dst + c);
            }
            if (lane == 0) a.scale[row[u] * a.scale_row + run[u] * a.scale_run] = r.scale;
        }
    }
}

// Runs too long for registers: a workgroup per run, read twice.
template <typename T>
__global__ __launch_bounds__(256) void pack_long_kernel(const PackArgs a) {
    __shared__ uint32_t part[4];
    for (uint32_t id = blockIdx.x; id < a.total; id += gridDim.x) {
        const uint32_t rw = a.groups.div(id);
        const int64_t row = rw;
        const int col = static_cast<int>(id - rw * a.groups.d) * a.group;
        const int len = a.cols - col < a.group ? a.cols - col : a.group;
        const T* src = static_cast<const T*>(a.x) + row * a.ldx + col;
        uint32_t t = 0;
        for (int c = threadIdx.x; c < len; c += 256) {
            const uint32_t b = __float_as_uint(widen(src[c])) & 0x7fffffffu;
            t = b > t ? b : t;
        }
        t = lanes_umax(t, kWave);
        __syncthreads();  // the previous run's maxima have been read
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = t;
        __syncthreads();
        t = part[0];
        for (int i = 1; i < 4; ++i) t = part[i] > t ? part[i] : t;
        const RunScale r = run_scale(t);
        int8_t* dst = a.q + row * a.ldq + col;
        for (int c = threadIdx.x; c < len; c += 256)
            dst[c] = static_cast<int8_t>(t >= 0x7f800000u ? 0 : run_quant(widen(src[c]), r));
        if (threadIdx.x == 0) a.scale[row * a.scale_row + (id - rw * a.groups.d) * a.scale_run] = r.scale;
    }
}

struct UnpackArgs {
    const int8_t* q;
    const float* scale;
    void* x;
    int64_t ldx, ldq;
    uint32_t total;  // pieces of VEC elements of this launch
    int groups;
    FastDiv per_row, per_group;  // pieces
};

template <typename T, int VEC, int UN>
__global__ __launch_bounds__(256) void unpack_kernel(const UnpackArgs a) {
    const uint32_t stride = gridDim.x * 256;
    for (uint32_t first = blockIdx.x * 256 + threadIdx.x; first < a.total; first += stride * UN) {
        Pack<int8_t, VEC> in[UN];
        float s[UN];
        int64_t to[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            uint32_t id = first + u * stride;
            id = id < a.total ? id : a.total - 1;
            const uint32_t row = a.per_row.div(id);
            const uint32_t piece = id - row * a.per_row.d;
            in[u].load(a.q + static_cast<int64_t>(row) * a.ldq + piece * VEC);
            s[u] = a.scale[static_cast<int64_t>(row) * a.groups + a.per_group.div(piece)];
            to[u] = static_cast<int64_t>(row) * a.ldx + piece * VEC;
        }
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            if (first + u * stride >= a.total) continue;
            float v[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                v[j] = in[u].get(j) * s[u];
                // the fp32 product is the value; without this the compiler forms fp16 results with one mixed-precision
                // instruction, rounding the exact product where the other types round the fp32 one
                asm("" : "+v"(v[j]));
            }
            Pack<T, VEC> o;
            o.set_all(v);
            o.store(static_cast<T*>(a.x) + to[u]);
        }
    }
}

// The widest piece that every row start, run start and run end is a multiple of (the last run of a row ends at cols).
static int piece_of(const void* x, int dtype, int64_t cols, int64_t ldx, int64_t group, const void* q, int64_t ldq) {
    const int64_t size = element_size(dtype);
    for (int vec = size == 4 ? 4 : 8; vec > 1; vec >>= 1) {
        const bool runs = group >= cols || group % vec == 0;
        if (runs && cols % vec == 0 && ldx % vec == 0 && ldq % vec == 0 && aligned_to(x, vec * size) && aligned_to(q, vec))
            return vec;
    }
    return 1;
}

template <typename T, int VEC>
static void launch_pack_vec(PackArgs& a, hipStream_t s) {
    const int64_t run = a.group < a.cols ? a.group : a.cols;
    const int64_t pieces = ceil_div(run, VEC);
    a.lanes = 1;
    while (a.lanes < kWave && a.lanes < pieces) a.lanes <<= 1;
    const int64_t per_lane = ceil_div(pieces, a.lanes);
    const int blocks = grid_for(a.total, 256 / a.lanes);
    if (per_lane <= 1)
        hipLaunchKernelGGL((pack_kernel<T, VEC, 1, 4>), dim3(grid_for(ceil_div(a.total, 4), 256 / a.lanes)), dim3(256), 0, s, a);
    else if (per_lane <= 2)
        hipLaunchKernelGGL((pack_kernel<T, VEC, 2, 2>), dim3(grid_for(ceil_div(a.total, 2), 256 / a.lanes)), dim3(256), 0, s, a);
    else if (per_lane <= 4)
        hipLaunchKernelGGL((pack_kernel<T, VEC, 4, 1>), dim3(blocks), dim3(256), 0, s, a);
    else if (per_lane <= 8)
        hipLaunchKernelGGL((pack_kernel<T, VEC, 8, 1>), dim3(blocks), dim3(256), 0, s, a);
    else if (per_lane <= 16)
        hipLaunchKernelGGL((pack_kernel<T, VEC, 16, 1>), dim3(blocks), dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((pack_long_kernel<T>), dim3(a.total < 2048 ? a.total : 2048), dim3(256), 0, s, a);
}

template <typename T>
static void launch_pack(PackArgs& a, int vec, hipStream_t s) {
    if constexpr (sizeof(T) == 2) {
        if (vec == 8) return launch_pack_vec<T, 8>(a, s);
    }
    if (vec == 4) return launch_pack_vec<T, 4>(a, s);
    if (vec == 2) return launch_pack_vec<T, 2>(a, s);
    launch_pack_vec<T, 1>(a, s);
}

template <typename T, int VEC>
static void launch_unpack_vec(const UnpackArgs& a, hipStream_t s) {
    hipLaunchKernelGGL((unpack_kernel<T, VEC, 4>), dim3(grid_for(ceil_div(a.total, 4), 256)), dim3(256), 0, s, a);
}

template <typename T>
static void launch_unpack(const UnpackArgs& a, int vec, hipStream_t s) {
    if constexpr (sizeof(T) == 2) {
        if (vec == 8) return launch_unpack_vec<T, 8>(a, s);
    }
    if (vec == 4) return launch_unpack_vec<T, 4>(a, s);
    if (vec == 2) return launch_unpack_vec<T, 2>(a, s);
    launch_unpack_vec<T, 1>(a, s);
}

static int check_pack(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, int64_t group, const void* q,
                      int64_t ldq, const void* scale) {
    if (!float_type(dtype)) return TANGO_ERR_UNSUPPORTED;
    if (rows < 0 || cols < 0 || group <= 0) return TANGO_ERR_INVALID_ARG;
    if (rows == 0 || cols == 0) return TANGO_OK;
    if (!x || !q || !scale || ldx < 0 || ldq < 0 || !aligned_to(x, element_size(dtype)) || !aligned_to(scale, 4))
        return TANGO_ERR_INVALID_ARG;
    if (cols >= (1LL << 30)) return TANGO_ERR_UNSUPPORTED;
    return TANGO_OK;
}

}  // namespace tango

using namespace tango;

extern "C" {

int tango_pack_i8(int8_t* q, int64_t ldq, float* scale, int64_t scale_row, int64_t scale_run, const void* x, int dtype,
                  int64_t rows, int64_t cols, int64_t ldx, int64_t group, tango_stream_t stream) {
    const int rc = check_pack(x, dtype, rows, cols, ldx, group, q, ldq, scale);
    if (rc != TANGO_OK || rows == 0 || cols == 0) return rc;
    if (rows > 1 && ldq < cols) return TANGO_ERR_INVALID_ARG;  // rows of the result would overlap
    if (scale_row < 0 || scale_run < 0) return TANGO_ERR_INVALID_ARG;
    if (group > cols) group = cols;
    const int64_t groups = ceil_div(cols, group);
    const int vec = piece_of(x, dtype, cols, ldx, group, q, ldq);
    const int64_t slab = ((1LL << 30) / groups) > 0 ? (1LL << 30) / groups : 1;  // runs of a launch stay below 2^31
    for (int64_t r0 = 0; r0 < rows; r0 += slab) {
        PackArgs a;
        a.rows = rows - r0 < slab ? rows - r0 : slab;
        a.x = static_cast<const char*>(x) + r0 * ldx * element_size(dtype);
        a.q = q + r0 * ldq;
        a.scale = scale + r0 * scale_row;
        a.scale_row = scale_row;
        a.scale_run = scale_run;
        a.ldx = ldx;
        a.ldq = ldq;
        a.total = static_cast<uint32_t>(a.rows * groups);
        a.cols = static_cast<int>(cols);
        a.group = static_cast<int>(group);
        a.groups = FastDiv(static_cast<uint32_t>(groups));
        if (dtype == TANGO_F32)
            launch_pack<float>(a, vec, as_stream(stream));
        else if (dtype == TANGO_BF16)
            launch_pack<bf16_t>(a, vec, as_stream(stream));
        else
            launch_pack<f16_t>(a, vec, as_stream(stream));
        if (launch_status() != TANGO_OK) return TANGO_ERR_LAUNCH;
    }
    return TANGO_OK;
}

int tango_unpack_i8(void* x, int dtype, int64_t ldx, const int8_t* q, int64_t ldq, const float* scale, int64_t rows,
                    int64_t cols, int64_t group, tango_stream_t stream) {
    const int rc = check_pack(x, dtype, rows, cols, ldx, group, q, ldq, scale);
    if (rc != TANGO_OK || rows == 0 || cols == 0) return rc;
    if (rows > 1 && ldx < cols) return TANGO_ERR_INVALID_ARG;
    if (group > cols) group = cols;
    const int64_t groups = ceil_div(cols, group);
    const int vec = piece_of(x, dtype, cols, ldx, group, q, ldq);
    const int64_t pieces = cols / vec;
    const int64_t slab = ((1LL << 30) / pieces) > 0 ? (1LL << 30) / pieces : 1;
    for (int64_t r0 = 0; r0 < rows; r0 += slab) {
        const int64_t n = rows - r0 < slab ? rows - r0 : slab;
        UnpackArgs a;
        a.q = q + r0 * ldq;
        a.scale = scale + r0 * groups;
        a.x = static_cast<char*>(x) + r0 * ldx * element_size(dtype);
        a.ldx = ldx;
        a.ldq = ldq;
        a.total = static_cast<uint32_t>(n * pieces);
        a.groups = static_cast<int>(groups);
        a.per_row = FastDiv(static_cast<uint32_t>(pieces));
        a.per_group = FastDiv(static_cast<uint32_t>(group >= cols ? pieces : group / vec));
        if (dtype == TANGO_F32)
            launch_unpack<float>(a, vec, as_stream(stream));
        else if (dtype == TANGO_BF16)
            launch_unpack<bf16_t>(a, vec, as_stream(stream));
        else
            launch_unpack<f16_t>(a, vec, as_stream(stream));
        if (launch_status() != TANGO_OK) return TANGO_ERR_LAUNCH;
    }
    return TANGO_OK;
}

}  // extern "C"
