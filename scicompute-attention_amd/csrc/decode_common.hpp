// Shared pieces of the decode kernels over 16/32-bit pages (decode.hip) and over 8-bit pages
// (decode8.hip): element traits, MFMA wrappers, the split range and the log-sum-exp combine.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "sca_device.hpp"

namespace sca_hip {
namespace {

constexpr int kDecodeThreads = 256;
constexpr int kDecodeWaves = kDecodeThreads / kWave;

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2v __attribute__((ext_vector_type(2)));

// ---- element traits --------------------------------------------------------------------------
// VE elements per 16-byte lane vector; dot4() accumulates the 16-byte product q.k into acc.
struct DecF16 {
    static constexpr int VE = 8;
    static __device__ __forceinline__ float dot(const uint4& q, const uint4& k, float acc) {
        acc = __builtin_amdgcn_fdot2(__builtin_bit_cast(half2v, q.x), __builtin_bit_cast(half2v, k.x),
                                     acc, false);
        acc = __builtin_amdgcn_fdot2(__builtin_bit_cast(half2v, q.y), __builtin_bit_cast(half2v, k.y),
                                     acc, false);
        acc = __builtin_amdgcn_fdot2(__builtin_bit_cast(half2v, q.z), __builtin_bit_cast(half2v, k.z),
                                     acc, false);
        acc = __builtin_amdgcn_fdot2(__builtin_bit_cast(half2v, q.w), __builtin_bit_cast(half2v, k.w),
                                     acc, false);
        return acc;
    }
    static __device__ __forceinline__ void unpack(const uint4& raw, float* out) {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            out[2 * i] = F16::to_float(static_cast<uint16_t>(w[i] & 0xffffu));
            out[2 * i + 1] = F16::to_float(static_cast<uint16_t>(w[i] >> 16));
        }
    }
    static __device__ __forceinline__ void store(void* dst, const float* v) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = static_cast<uint32_t>(F16::from_float(v[2 * i])) |
                   (static_cast<uint32_t>(F16::from_float(v[2 * i + 1])) << 16);
        }
        *static_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ void store1(uint8_t* row, int d, float v) {
        reinterpret_cast<uint16_t*>(row)[d] = F16::from_float(v);
    }
};

struct DecBF16 {
    static constexpr int VE = 8;
    static __device__ __forceinline__ float dot(const uint4& q, const uint4& k, float acc) {
        acc = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2v, q.x),
                                              __builtin_bit_cast(bf16x2v, k.x), acc, false);
        acc = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2v, q.y),
                                              __builtin_bit_cast(bf16x2v, k.y), acc, false);
        acc = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2v, q.z),
                                              __builtin_bit_cast(bf16x2v, k.z), acc, false);
        acc = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2v, q.w),
                                              __builtin_bit_cast(bf16x2v, k.w), acc, false);
        return acc;
    }
    static __device__ __forceinline__ void unpack(const uint4& raw, float* out) {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            out[2 * i] = __builtin_bit_cast(float, w[i] << 16);
            out[2 * i + 1] = __builtin_bit_cast(float, w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ void store(void* dst, const float* v) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = static_cast<uint32_t>(BF16::from_float(v[2 * i])) |
                   (static_cast<uint32_t>(BF16::from_float(v[2 * i + 1])) << 16);
        }
        *static_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ void store1(uint8_t* row, int d, float v) {
        reinterpret_cast<uint16_t*>(row)[d] = BF16::from_float(v);
    }
};

struct DecF32 {
    static constexpr int VE = 4;
    static __device__ __forceinline__ float dot(const uint4& q, const uint4& k, float acc) {
        acc = fmaf(__builtin_bit_cast(float, q.x), __builtin_bit_cast(float, k.x), acc);
        acc = fmaf(__builtin_bit_cast(float, q.y), __builtin_bit_cast(float, k.y), acc);
        acc = fmaf(__builtin_bit_cast(float, q.z), __builtin_bit_cast(float, k.z), acc);
        acc = fmaf(__builtin_bit_cast(float, q.w), __builtin_bit_cast(float, k.w), acc);
        return acc;
    }
    static __device__ __forceinline__ void unpack(const uint4& raw, float* out) {
        out[0] = __builtin_bit_cast(float, raw.x);
        out[1] = __builtin_bit_cast(float, raw.y);
        out[2] = __builtin_bit_cast(float, raw.z);
        out[3] = __builtin_bit_cast(float, raw.w);
    }
    static __device__ __forceinline__ void store(void* dst, const float* v) {
        *static_cast<uint4*>(dst) =
            make_uint4(__builtin_bit_cast(uint32_t, v[0]), __builtin_bit_cast(uint32_t, v[1]),
                       __builtin_bit_cast(uint32_t, v[2]), __builtin_bit_cast(uint32_t, v[3]));
    }
    static __device__ __forceinline__ void store1(uint8_t* row, int d, float v) {
        reinterpret_cast<float*>(row)[d] = v;
    }
};

// Keys per split, ceil(len / splits).
__device__ __forceinline__ int64_t SplitChunk(int64_t len, int64_t splits) {
    if (len <= 0) return 0;
    if (len < (int64_t{1} << 31)) {
        return (static_cast<uint32_t>(len) + static_cast<uint32_t>(splits) - 1) /
               static_cast<uint32_t>(splits);
    }
    return (len + splits - 1) / splits;
}

// Split merge (reference decode_splitk.cu:143-182): out = sum_s O_s e^{m_s - m*} / sum_s l_s e^{m_s - m*},
// with m* = max_s m_s, splits with m_s = -inf skipped and out = 0 when the denominator is 0.
// One thread per (b, h_q, 4 consecutive d): the split loads of a thread are independent, so
// they overlap instead of forming a chain, and neighbouring threads read neighbouring bytes.
constexpr int kCombineThreads = 256;

template <typename E, int D>
__global__ __launch_bounds__(kCombineThreads) void decode_combine_kernel(const sca_decode_params p) {
    constexpr int64_t kElemBytes = 16 / E::VE;
    constexpr int kQuads = D / 4;
    // batch * heads fits 32 bits (each is below 2^16); kQuads is a constant.
    const int64_t first = static_cast<int64_t>(blockIdx.x) * kCombineThreads;
    const int64_t first_row = first / kQuads;
    const uint32_t within = static_cast<uint32_t>(first - first_row * kQuads) + threadIdx.x;
    const int64_t flat_bh = first_row + within / kQuads;
    if (flat_bh >= p.batch * p.num_heads) return;
    const int d0 = static_cast<int>(within % kQuads) * 4;
    const int64_t b = static_cast<uint32_t>(flat_bh) / static_cast<uint32_t>(p.num_heads);
    const int64_t h = static_cast<uint32_t>(flat_bh) % static_cast<uint32_t>(p.num_heads);
    const int ns = static_cast<int>(p.num_splits);
    const float* pm = p.partial_m + flat_bh * ns;
    const float* pl = p.partial_l + flat_bh * ns;
    const float* po = p.partial_o + flat_bh * ns * D + d0;

    float m_all = neg_inf();
#pragma unroll 8
    for (int s = 0; s < ns; ++s) m_all = fmaxf(m_all, pm[s]);
    float l_all = 0.0f;
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int s = 0; s < ns; ++s) {
        const float ms = pm[s];
        const float w = (ms == neg_inf()) ? 0.0f : fast_exp2((ms - m_all) * kLog2e);
        l_all = fmaf(pl[s], w, l_all);
        const float* o = po + static_cast<int64_t>(s) * D;
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = fmaf(o[i], w, acc[i]);
    }
    const float inv = l_all > 0.0f ? 1.0f / l_all : 0.0f;
    uint8_t* out_row = static_cast<uint8_t*>(p.out) + (b * p.o_sb + h * p.o_sh) * kElemBytes;
#pragma unroll
    for (int i = 0; i < 4; ++i) E::store1(out_row, d0 + i, acc[i] * inv);
}

constexpr int kRankBatch = 256;  // ragged batches up to this size are ranked in the kernel

constexpr int kMfmaTile = 32;   // tokens per wave iteration
constexpr int kMfmaHeads = 16;  // query heads per workgroup (MFMA N)

template <typename E>
struct DecMfma;

template <>
struct DecMfma<DecF16> {
    using vec8 = half8;
    using Tr = TrRead<F16>;
    typedef _Float16 pair_t __attribute__((ext_vector_type(2)));
    static __device__ __forceinline__ floatx4 mma(const vec8& a, const vec8& b, floatx4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        typedef float f2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){a, b}, pair_t));
    }
    // Weights from kSplitLeast on, times kScale, have all their 24 bits above fp16's smallest value.
    static constexpr float kScale = 0x1p15f;
    static constexpr float kSplitLeast = 0x1p-14f;
    // Two weights (scaled) as fp16 pairs hi + mid + lo, each rounded towards zero, mid and lo at least
    // 2^-24 (2^-25 of the smallest weight).
    static __device__ __forceinline__ void split3(float a, float b, uint32_t* w) {
        float ra = a, rb = b;
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            const auto pair = __builtin_amdgcn_cvt_pkrtz(ra, rb);
            w[i] = __builtin_bit_cast(uint32_t, pair);
            ra = fmaxf(ra - static_cast<float>(pair[0]), 0x1p-24f);
            rb = fmaxf(rb - static_cast<float>(pair[1]), 0x1p-24f);
        }
    }
};

template <>
struct DecMfma<DecBF16> {
    using vec8 = bf16x8;
    using Tr = TrRead<BF16>;
    typedef __bf16 pair_t __attribute__((ext_vector_type(2)));
    static __device__ __forceinline__ floatx4 mma(const vec8& a, const vec8& b, floatx4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        typedef float f2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){a, b}, pair_t));
    }
    static constexpr float kScale = 1.0f;
    static constexpr float kSplitLeast = 0.0f;  // bf16 has fp32's range
    // Two weights as bf16 pairs hi + mid + lo (8 bits each, by truncation), mid and lo at least 2^-126
    // unless the weight is 0.
    static __device__ __forceinline__ void split3(float a, float b, uint32_t* w) {
        float ra = a, rb = b;
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            const uint32_t ua = __builtin_bit_cast(uint32_t, ra), ub = __builtin_bit_cast(uint32_t, rb);
            w[i] = (ua >> 16) | (ub & 0xffff0000u);
            ra = __builtin_amdgcn_fmed3f(ra - __builtin_bit_cast(float, ua & 0xffff0000u), 0x1p-126f, a);
            rb = __builtin_amdgcn_fmed3f(rb - __builtin_bit_cast(float, ub & 0xffff0000u), 0x1p-126f, b);
        }
    }
};

// 32-byte segment swizzle of V row t, so that the 8 rows one half of a transposed read touches land on
// distinct segments of the 256-byte bank window: a row is D/16 segments, so rows of 0 mod 8 segments
// all start alike, of 4 mod 8 every other one, and of 2 or 6 mod 8 every fourth. (Rows t and t + 16
// share it, which the two transposed reads of a lane rely on.)
template <int D>
__device__ __forceinline__ int VSwz(int t) {
    constexpr int kStart = (D / 16) % 8;
    return kStart == 0 ? (t & 7) : kStart == 4 ? ((t >> 1) & 3) : ((t >> 2) & 1);
}

bool Aligned16(const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0; }

}  // namespace
}  // namespace sca_hip
