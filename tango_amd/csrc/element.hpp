// Element types of the operators that take fp32, bf16 and fp16 tensors: widening loads and once-rounded stores.
#pragma once
#include "common.hpp"

namespace tango {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// A lane's VEC consecutive elements as 32-bit words, loaded by the widest instructions that VEC allows.
template <typename T, int VEC>
struct Pack {
    static constexpr int kBytes = VEC * static_cast<int>(sizeof(T));
    static constexpr int kWords = (kBytes + 3) / 4;
    uint32_t w[kWords];

    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0;
    }
    // p at any multiple of an element: global memory takes vector accesses at any address
    __device__ __forceinline__ void load_any(const T* p) {
        static_assert(kBytes == 4 || kBytes == 8 || kBytes % 16 == 0, "whole vectors");
        if constexpr (kBytes == 4) {
            typedef uint32_t U __attribute__((aligned(1)));
            w[0] = *reinterpret_cast<const U*>(p);
        } else if constexpr (kBytes == 8) {
            typedef u32x2 U __attribute__((aligned(1)));
            const u32x2 t = *reinterpret_cast<const U*>(p);
            w[0] = t[0];
            w[1] = t[1];
        } else {
            typedef u32x4 U __attribute__((aligned(1)));
#pragma unroll
            for (int i = 0; i < kBytes / 16; ++i) {
                const u32x4 t = reinterpret_cast<const U*>(p)[i];
#pragma unroll
                for (int j = 0; j < 4; ++j) w[4 * i + j] = t[j];
            }
        }
    }
    __device__ __forceinline__ void store_any(T* p) const {
        static_assert(kBytes == 4 || kBytes == 8 || kBytes % 16 == 0, "whole vectors");
        if constexpr (kBytes == 4) {
            typedef uint32_t U __attribute__((aligned(1)));
            *reinterpret_cast<U*>(p) = w[0];
        } else if constexpr (kBytes == 8) {
            typedef u32x2 U __attribute__((aligned(1)));
            u32x2 t;
            t[0] = w[0];
            t[1] = w[1];
            *reinterpret_cast<U*>(p) = t;
        } else {
            typedef u32x4 U __attribute__((aligned(1)));
#pragma unroll
            for (int i = 0; i < kBytes / 16; ++i) {
                u32x4 t;
#pragma unroll
                for (int j = 0; j < 4; ++j) t[j] = w[4 * i + j];
                reinterpret_cast<U*>(p)[i] = t;
            }
        }
    }
    // The first n elements (n < VEC), the others zero; one access each.
    __device__ __forceinline__ void load_some(const T* p, int n) {
        constexpr int kBits = 8 * static_cast<int>(sizeof(T));
        zero();
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (i < n) {
                uint32_t one;
                if constexpr (sizeof(T) == 4) one = *reinterpret_cast<const uint32_t*>(p + i);
                if constexpr (sizeof(T) == 2) one = *reinterpret_cast<const uint16_t*>(p + i);
                if constexpr (sizeof(T) == 1) one = *reinterpret_cast<const uint8_t*>(p + i);
                w[i * kBits / 32] |= one << (i * kBits % 32);
            }
    }
    __device__ __forceinline__ void store_some(T* p, int n) const {
        constexpr int kBits = 8 * static_cast<int>(sizeof(T));
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (i < n) {
                const uint32_t one = w[i * kBits / 32] >> (i * kBits % 32);
                if constexpr (sizeof(T) == 4) *reinterpret_cast<uint32_t*>(p + i) = one;
                if constexpr (sizeof(T) == 2) *reinterpret_cast<uint16_t*>(p + i) = static_cast<uint16_t>(one);
                if constexpr (sizeof(T) == 1) *reinterpret_cast<uint8_t*>(p + i) = static_cast<uint8_t>(one);
            }
    }
    // p aligned to min(kBytes, 16)
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (kBytes >= 16) {
            const u32x4* v = reinterpret_cast<const u32x4*>(p);
#pragma unroll
            for (int i = 0; i < kBytes / 16; ++i) {
                const u32x4 t = v[i];
#pragma unroll
                for (int j = 0; j < 4; ++j) w[4 * i + j] = t[j];
            }
        } else if constexpr (kBytes == 8) {
            const u32x2 t = *reinterpret_cast<const u32x2*>(p);
            w[0] = t[0];
            w[1] = t[1];
        } else if constexpr (kBytes == 4) {
            w[0] = *reinterpret_cast<const uint32_t*>(p);
        } else if constexpr (kBytes == 2) {
            w[0] = *reinterpret_cast<const uint16_t*>(p);
        } else {
            w[0] = *reinterpret_cast<const uint8_t*>(p);
        }
    }
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (kBytes >= 16) {
            u32x4* v = reinterpret_cast<u32x4*>(p);
#pragma unroll
            for (int i = 0; i < kBytes / 16; ++i) {
                u32x4 t;
#pragma unroll
                for (int j = 0; j < 4; ++j) t[j] = w[4 * i + j];
                v[i] = t;
            }
        } else if constexpr (kBytes == 8) {
            u32x2 t;
            t[0] = w[0];
            t[1] = w[1];
            *reinterpret_cast<u32x2*>(p) = t;
        } else if constexpr (kBytes == 4) {
            *reinterpret_cast<uint32_t*>(p) = w[0];
        } else if constexpr (kBytes == 2) {
            *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(w[0]);
        } else {
            *reinterpret_cast<uint8_t*>(p) = static_cast<uint8_t>(w[0]);
        }
    }
    // i a compile-time constant after unrolling
    __device__ __forceinline__ float get(int i) const {
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(w[i]);
        } else if constexpr (sizeof(T) == 1) {
            return static_cast<float>(static_cast<int8_t>(w[i / 4] >> (8 * (i & 3))));
        } else {
            const uint32_t u = w[i / 2];
            if constexpr (__is_same(T, bf16_t)) return __uint_as_float((i & 1) ? (u & 0xffff0000u) : (u << 16));
            const uint16_t h = static_cast<uint16_t>((i & 1) ? (u >> 16) : u);
            return static_cast<float>(__builtin_bit_cast(f16_t, h));
        }
    }
    __device__ __forceinline__ void set_all(const float* v) {  // one rounding, to nearest even
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) w[i] = __float_as_uint(v[i]);
        } else {
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                const uint32_t lo = __builtin_bit_cast(uint16_t, static_cast<T>(v[2 * i]));
                const uint32_t hi = 2 * i + 1 < VEC ? __builtin_bit_cast(uint16_t, static_cast<T>(v[2 * i + 1])) : 0;
                w[i] = lo | (hi << 16);
            }
        }
    }
};

template <typename T>
__device__ __forceinline__ float widen(T v) {
    return static_cast<float>(v);
}

// x / d for 0 <= x < 2^31 and a divisor known on the host: one high product and a shift (the multiplier is
// ceil(2^(32+s) / d) with s = ceil(log2 d) - 1, exact for 31-bit x by the round-up method of Granlund and Montgomery).
struct FastDiv {
    uint32_t d, mul, shift;
    FastDiv() = default;
    explicit FastDiv(uint32_t div) : d(div), mul(0), shift(0) {
        if (div > 1) {
            while ((1ull << (shift + 1)) < div) ++shift;  // shift = ceil(log2 div) - 1
            mul = static_cast<uint32_t>(((1ull << (32 + shift)) + div - 1) / div);
        }
    }
    __device__ __forceinline__ uint32_t div(uint32_t x) const { return d > 1 ? __umulhi(x, mul) >> shift : x; }
};

inline bool aligned_to(const void* p, int64_t bytes) { return (reinterpret_cast<uintptr_t>(p) % bytes) == 0; }

inline int element_size(int dtype) { return dtype == TANGO_F32 ? 4 : 2; }
inline bool float_type(int dtype) { return dtype == TANGO_F32 || dtype == TANGO_BF16 || dtype == TANGO_F16; }

}  // namespace tango
