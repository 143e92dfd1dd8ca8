// What the device sources of the output unit, the losses and the checkpoints
// share: vector types, the 16-bit formats, matrix products of 16 x 16 x 32, and
// the host side's checks.

#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr int kGroup = 8;   // 16-bit elements per 128-bit access

// 16-bit formats: a pair in a 32-bit word <-> two floats.  The conversions
// back round to nearest even (v_cvt_pk_bf16_f32, v_cvt_f16_f32), as torch's.
struct Bf16 {
    static constexpr uint32_t kNegInf2 = 0xFF80FF80u;
    static constexpr uint32_t kNegInf = 0xFF80u;
    static constexpr uint32_t kNan2 = 0x7FC07FC0u;
    __device__ static float lo(uint32_t w) { return __uint_as_float(w << 16); }
    __device__ static float hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
    __device__ static uint32_t pack(float a, float b) {
        const f32x2 f = {a, b};
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, bf16x2));
    }
};
struct F16 {
    static constexpr uint32_t kNegInf2 = 0xFC00FC00u;
    static constexpr uint32_t kNegInf = 0xFC00u;
    static constexpr uint32_t kNan2 = 0x7E007E00u;
    __device__ static float lo(uint32_t w) { return float(__builtin_bit_cast(f16x2, w).x); }
    __device__ static float hi(uint32_t w) { return float(__builtin_bit_cast(f16x2, w).y); }
    __device__ static uint32_t pack(float a, float b) {
        const f32x2 f = {a, b};
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, f16x2));
    }
};

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLog2eLo = 1.92596299e-8f;   // log2(e) - kLog2e

// exp(t) for t <= 0 as 2^(t log2 e), the product rounded: relative error up to
// |t| 2^-24 and no subnormal results.  For the terms of a row's sum alone:
// against the lane's own maximum |t| is small, and the sum's logarithm comes
// out as close to 64 bits as with expf (mean relative error of the row losses
// 3.3e-8 | 3.9e-8 at 4092 x 128256, 3.8e-8 | 4.2e-8 at 510 x 4096).
__device__ __forceinline__ float exp_term(float t) { return __builtin_amdgcn_exp2f(t * kLog2e); }

// exp(t) for finite t <= 0 or so and t = -inf, to an ulp or two, subnormal
// results included: 2^n times 2^f, f the rest of t log2 e in two parts.  What
// becomes a probability takes this one: with exp_term 1.1e-4 of the bf16
// results at 4092 x 128256 were not the nearest to the exact ones, with it
// 0.4e-4 to 0.9e-4, as with expf, which needs 5 instructions more.  us with
// exp_term | this, bf16 rows: 4092 x 128256 403 | 427, 4092 x 32000 80 | 83,
// 1023 x 50257 47 | 51, 20000 x 4096 49 | 54.
__device__ __forceinline__ float exp_full(float t) {
    t = fmaxf(t, -200.0f);   // 2^f of an infinite t would be NaN
    const float n = rintf(t * kLog2e);
    return __builtin_amdgcn_ldexpf(__builtin_amdgcn_exp2f(fmaf(t, kLog2eLo, fmaf(t, kLog2e, -n))), int(n));
}

// A partial logsumexp: the maximum so far and the sum of exp(x - base(max)).
// base() is the maximum itself, or 0 where that is infinite, so that rows
// with infinities give what logsumexp gives: +inf, or -inf for a row of them.
struct Lse {
    float m, s;
};
__device__ __forceinline__ float base(float m) { return __builtin_isinf(m) ? 0.0f : m; }

// The same over groups of kN neighbouring lanes of a wave, in every lane: the
// maximum first, so that each lane rescales its part once (merging pairs costs
// two exponentials a step: 300,000 rows of 2000 bf16 1,030 us, so 694), then the
// sums.
template <int kN>
__device__ __forceinline__ Lse lane_lse(Lse p) {
    float m = p.m;
#pragma unroll
    for (int d = kN / 2; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
    // an empty part stays empty whatever the bases are; a NaN sum stays NaN
    float s = p.s == 0.0f ? 0.0f : p.s * expf(base(p.m) - base(m));
#pragma unroll
    for (int d = kN / 2; d > 0; d >>= 1) s += __shfl_xor(s, d);
    return {m, s};
}

// logsumexp over a row's kT lanes, the same value in every one: in one wave
// without a barrier, else through LDS.
template <int kT>
__device__ __forceinline__ float block_lse(Lse p, Lse* parts) {
    p = lane_lse<(kT < 64 ? kT : 64)>(p);
    if constexpr (kT > 64) {
        if ((threadIdx.x & 63) == 0) parts[threadIdx.x >> 6] = p;
        __syncthreads();
        p = lane_lse<kT / 64>(parts[threadIdx.x % (kT / 64)]);
    }
    return base(p.m) + logf(p.s);
}

// Rows of one workgroup: rows that one wave or less reads share it.
template <int kT>
constexpr int kRowsOf = kT <= 64 ? 256 / kT : 1;

// What a row's label asks for.
enum RowKind { kValid, kIgnored, kBadLabel };
__device__ __forceinline__ RowKind row_kind(int64_t y, int64_t ignore_index, uint32_t vocab) {
    if (y == ignore_index) return kIgnored;
    return (y < 0 || y >= int64_t(vocab)) ? kBadLabel : kValid;
}

// Products of 16 x 16 x 32: operand lanes hold row or column l % 16, terms 8
// (l / 16) to + 7; result lanes column l % 16, rows 4 (l / 16) to + 3.
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ f32x4 mfma(Bf16, u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
}
__device__ __forceinline__ f32x4 mfma(F16, u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
}

inline int status() {
    // the runtime keeps a failed launch as the thread's last error: reading it clears it
    return int(hipGetLastError());
}

inline bool misaligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }

// Lanes of one launch: a dispatch takes fewer than 2^32 along a dimension.
constexpr uint64_t kMaxLanes = uint64_t(1) << 31;

}  // namespace
