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
    float top, inv, rec;  // the maximum scaled to [0.5, 1); 127 / top; 1 / top
    float times;          // 127 times that power of two
    float scale;
    int exp;
    bool held, plain;     // finite and not zero; and in a range where nothing below over- or underflows
};

__device__ __forceinline__ RunScale run_scale(uint32_t top_bits) {
    RunScale r;
    const float top = __uint_as_float(top_bits);
    r.held = top_bits != 0 && top_bits < 0x7f800000u;
    r.exp = __builtin_amdgcn_frexp_expf(r.held ? top : 1.0f);
    r.top = __builtin_amdgcn_ldexpf(r.held ? top : 1.0f, -r.exp);
    r.inv = 127.0f / r.top;
    r.rec = 1.0f / r.top;
    r.plain = r.held && r.exp > -100 && r.exp < 100;
    r.times = __builtin_amdgcn_ldexpf(127.0f, r.plain ? -r.exp : 0);
    r.scale = r.held ? fminf(top / 127.0f, kLargestScale) : top_bits ? __uint_as_float(0x7fc00000u) : 0.0f;
    return r;
}

__device__ __forceinline__ int run_quant(float x, const RunScale& r) {
    const int n = nearest_127(__builtin_amdgcn_ldexpf(fabsf(x), -r.exp), r.top, r.inv);
    return !r.held ? 0 : x < 0.0f ? -n : n;
}

// The integers of VEC elements, four to a word.  16-bit elements: 127 x is exact in fp32, and a quotient refined by one
// step from a correctly rounded reciprocal is correctly rounded, so a tie, which is representable, is met exactly, and
// no other quotient of 16-bit numbers (11 bits at most) is closer to one than 2^-19 of itself; six instructions an element.  fp32 elements: the approximate
// quotient decides unless it is within 2^-14 of a tie (its error is below 2^-15); then nearest_127 does, for the whole
// piece.  Either way what is far from the ordinary range goes to nearest_127.
template <typename T, int VEC>
__device__ __forceinline__ void quant_piece(const Pack<T, VEC>& in, const RunScale& r, int (&n)[VEC]) {
    bool sure = r.plain;
    if constexpr (sizeof(T) == 4) {
        float far = 0.0f;
        const float inv = __builtin_amdgcn_ldexpf(r.inv, r.plain ? -r.exp : 0);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float y = in.get(j) * inv, k = rintf(y);
            far = fmaxf(far, fabsf(y - k));
            n[j] = static_cast<int>(k);
        }
        sure = sure && far < 0.5f - 0x1p-14f;
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float t = in.get(j) * r.times, y0 = t * r.rec;
            const float y = __builtin_fmaf(__builtin_fmaf(-y0, r.top, t), r.rec, y0);
            n[j] = static_cast<int>(rintf(y));
        }
    }
    if (!sure) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) n[j] = run_quant(in.get(j), r);
    }
}

// The largest |x| of VEC elements as the bits of an fp32 number (ordered like the numbers; a NaN is the largest).
template <typename T, int VEC, int R>
__device__ __forceinline__ uint32_t largest_bits(const Pack<T, VEC> (&in)[R]) {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    if constexpr (sizeof(T) == 4) {
        uint32_t t = 0;
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) t = __builtin_elementwise_max(t, in[i].w[j] & 0x7fffffffu);
        return t;
    } else {
        u16x2 t = {0, 0};
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int j = 0; j < Pack<T, VEC>::kWords; ++j)
                t = __builtin_elementwise_max(t, __builtin_bit_cast(u16x2, in[i].w[j] & 0x7fff7fffu));
        const uint16_t most = t[0] > t[1] ? t[0] : t[1];
        if constexpr (__is_same(T, bf16_t)) return static_cast<uint32_t>(most) << 16;
        return __float_as_uint(static_cast<float>(__builtin_bit_cast(f16_t, most)));
    }
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_umax(uint32_t v) {
    return __builtin_elementwise_max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xf, 0xf, true)));
}

// Maximum over `lanes` (a power of two, the same for the whole launch) neighbouring lanes, in all of them.
__device__ __forceinline__ uint32_t lanes_umax(uint32_t v, int lanes) {
    if (lanes >= 2) v = dpp_umax<0xb1>(v);
    if (lanes >= 4) v = dpp_umax<0x4e>(v);
    if (lanes >= 8) v = dpp_umax<0x141>(v);
    if (lanes >= 16) v = dpp_umax<0x140>(v);
    if (lanes >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = __builtin_elementwise_max(static_cast<uint32_t>(r[0]), static_cast<uint32_t>(r[1]));
    }
    if (lanes >= 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v = __builtin_elementwise_max(static_cast<uint32_t>(r[0]), static_cast<uint32_t>(r[1]));
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
                if constexpr (VEC == 1) {
                    if (c < len[u]) in[u][i].load(src + c);
                } else {
                    if (c + VEC <= len[u])
                        in[u][i].load_any(src + c);
                    else if (c < len[u])
                        in[u][i].load_some(src + c, len[u] - c);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < UN; ++u) top[u] = lanes_umax(largest_bits<T, VEC, R>(in[u]), a.lanes);
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
                int n[VEC];
                quant_piece<T, VEC>(in[u][i], r, n);
                if constexpr (VEC == 1) {
                    o.w[0] = static_cast<uint32_t>(n[0]) & 0xffu;
                } else {
#pragma unroll
                    for (int j = 0; j < VEC; j += 4) o.w[j / 4] = pack4(n[j], n[j + 1], n[j + 2], n[j + 3]);
                }
                if constexpr (VEC == 1) {
                    o.store(dst + c);
                } else {
                    if (c + VEC <= len[u])
                        o.store_any(dst + c);
                    else
                        o.store_some(dst + c, len[u] - c);
                }
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
            dst[c] = static_cast<int8_t>(run_quant(widen(src[c]), r));
        if (threadIdx.x == 0) a.scale[row * a.scale_row + (id - rw * a.groups.d) * a.scale_run] = r.scale;
    }
}

struct UnpackArgs {
    const int8_t* q;
    const float* scale;
    void* x;
    int64_t ldx, ldq;
    uint32_t total;  // pieces of VEC elements of this launch; every run has as many, the last ones of a short run are empty
    int cols, group;
    FastDiv groups, per_run;
};

template <typename T, int VEC, int UN>
__global__ __launch_bounds__(256) void unpack_kernel(const UnpackArgs a) {
    const uint32_t stride = gridDim.x * 256;
    for (uint32_t first = blockIdx.x * 256 + threadIdx.x; first < a.total; first += stride * UN) {
        Pack<int8_t, VEC> in[UN];
        float s[UN];
        int64_t to[UN];
        int left[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const bool ok = first + u * stride < a.total;
            const uint32_t id = ok ? first + u * stride : 0;
            const uint32_t run_id = a.per_run.div(id), row = a.groups.div(run_id);
            const int run = static_cast<int>(run_id - row * a.groups.d), at = static_cast<int>(id - run_id * a.per_run.d) * VEC;
            const int col = run * a.group + at;
            const int end = a.cols - run * a.group < a.group ? a.cols - run * a.group : a.group;
            left[u] = ok ? end - at : 0;
            const int8_t* p = a.q + static_cast<int64_t>(row) * a.ldq + col;
            in[u].zero();
            if constexpr (VEC == 1) {
                if (left[u] > 0) in[u].load(p);
            } else {
                if (left[u] >= VEC)
                    in[u].load_any(p);
                else if (left[u] > 0)
                    in[u].load_some(p, left[u]);
            }
            s[u] = a.scale[run_id];
            to[u] = static_cast<int64_t>(row) * a.ldx + col;
        }
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            if (left[u] <= 0) continue;
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
            T* p = static_cast<T*>(a.x) + to[u];
            if constexpr (VEC == 1) {
                o.store(p);
            } else {
                if (left[u] >= VEC)
                    o.store_any(p);
                else
                    o.store_some(p, left[u]);
            }
        }
    }
}

// Elements of a piece, at any alignment, the end of a run an element at a time; runs shorter than a piece altogether so.
// 16-bit types: 16 bytes ([232965, 602] bf16, whose rows start on multiples of four bytes: packed in 109 us, 142 us with
// pieces of four bytes).  fp32: 16 bytes restored, 32 packed where a run has them, so that 8 bytes are stored
// ([169343, 256] in runs of 32: 56 us against 59 us; restored with 32 bytes 37 us against 35 us).
static int piece_of(int dtype, int64_t cols, int64_t group, bool packing) {
    const int64_t run = group < cols ? group : cols;
    if (run >= 8 && (dtype != TANGO_F32 || packing)) return 8;
    return run >= 4 && dtype == TANGO_F32 ? 4 : 1;
}

template <typename T, int VEC, int R, int UN>
static void launch_pack_pieces(const PackArgs& a, hipStream_t s) {
    hipLaunchKernelGGL((pack_kernel<T, VEC, R, UN>), dim3(grid_for(ceil_div(a.total, UN), 256 / a.lanes)), dim3(256), 0, s, a);
}

template <typename T, int VEC>
static void launch_pack_vec(PackArgs& a, hipStream_t s) {
    const int64_t run = a.group < a.cols ? a.group : a.cols;
    const int64_t pieces = ceil_div(run, VEC);
    // lanes and pieces a lane with the fewest idle places (76 pieces: 16 lanes of 5; 64 lanes of 2 leave 52 of 128
    // places idle), the more lanes the better among equals
    int64_t best = 0, per_lane = 0;
    for (int lanes = kWave; lanes >= 1; lanes >>= 1) {
        const int64_t per = ceil_div(pieces, lanes);
        if (per > 8 || (best && per * lanes >= best)) continue;
        best = per * lanes;
        per_lane = per;
        a.lanes = lanes;
    }
    switch (per_lane) {
        case 1: return launch_pack_pieces<T, VEC, 1, 4>(a, s);
        case 2: return launch_pack_pieces<T, VEC, 2, 2>(a, s);
        case 3: return launch_pack_pieces<T, VEC, 3, 2>(a, s);
        case 4: return launch_pack_pieces<T, VEC, 4, 1>(a, s);
        case 5: return launch_pack_pieces<T, VEC, 5, 1>(a, s);
        case 6: return launch_pack_pieces<T, VEC, 6, 1>(a, s);
        case 7: return launch_pack_pieces<T, VEC, 7, 1>(a, s);
        case 8: return launch_pack_pieces<T, VEC, 8, 1>(a, s);
    }
    hipLaunchKernelGGL((pack_long_kernel<T>), dim3(a.total < 2048 ? a.total : 2048), dim3(256), 0, s, a);
}

template <typename T>
static void launch_pack(PackArgs& a, int vec, hipStream_t s) {
    if (vec == 8) return launch_pack_vec<T, 8>(a, s);
    if constexpr (sizeof(T) == 4) {
        if (vec == 4) return launch_pack_vec<T, 4>(a, s);
    }
    launch_pack_vec<T, 1>(a, s);
}

template <typename T>
static void launch_unpack(const UnpackArgs& a, int vec, hipStream_t s) {
    constexpr int kWide = 16 / static_cast<int>(sizeof(T));
    const dim3 grid(grid_for(ceil_div(a.total, 4), 256)), block(256);
    if (vec == 1)
        hipLaunchKernelGGL((unpack_kernel<T, 1, 4>), grid, block, 0, s, a);
    else
        hipLaunchKernelGGL((unpack_kernel<T, kWide, 4>), grid, block, 0, s, a);
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
    const int vec = piece_of(dtype, cols, group, true);
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
    const int vec = piece_of(dtype, cols, group, false);
    const int64_t per_run = ceil_div(group, vec), pieces = groups * per_run;  // of a row
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
        a.cols = static_cast<int>(cols);
        a.group = static_cast<int>(group);
        a.groups = FastDiv(static_cast<uint32_t>(groups));
        a.per_run = FastDiv(static_cast<uint32_t>(per_run));
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
