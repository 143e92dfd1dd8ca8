// Activation checkpoints in 8 bits for MI355X (gfx950): a decoder's input is
// packed in the forward pass and restored for its recompute in the backward.
//
// Blocks of 128 consecutive elements share a scale.  With a = max |x| of the
// block (at least 2^-100, so that its reciprocal stays finite) and T the
// largest code (127 of int8, 448 of fp8 e4m3):
//   code = round(x * (T / a)), restored = code * (a / T),
// both quotients rounded to fp32 and the codes to nearest even.  The error of
// an int8 element is at most a / 254 and a rounding; of an fp8 element 2^-4 of
// itself, or a 2^-10 / 448.  A block with an infinity or a NaN is restored as NaNs
// throughout: the step's loss shows them, as it does without the packing.
//
// Layout: the codes, 128 bytes a block (the last block's rest cleared), then
// the fp32 scales: 132 bytes a block in one run, so that one copy moves both.
//
// C ABI: include/slidefsdp.h.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/slidefsdp.h"
#include "sf_common.h"

namespace {

constexpr int kBlock = SF_ACT8_BLOCK;
// Elements of a lane.  Packing: one 128-bit access of codes, two of 16-bit
// elements.  Restoring: one 128-bit store of 16-bit elements, so that a wave's
// stores lie side by side (16 elements a lane, two stores with gaps: 16.8 M
// elements 11.6 | 9.3 us, 41.9 M 27.8 | 23.8).  Both move 51 MB at 16.8 M, in
// 9.8 and 9.7 us after each other, 5.2 TB/s (each repeated by itself 9.4 and 9.3);
// a device copy reaches 5.4.  Stores past the caches would take 8.2 us and cost the recompute that reads them next as much.
constexpr int kPack = 16;
constexpr int kUnpack = 8;
constexpr int kThreads = 256;
constexpr float kLeast = 0x1p-100f;
constexpr float kMost = 0x1.fffff0p127f;   // so that the largest code is not restored as infinity

struct Int8 {
    static constexpr float kTop = 127.0f;
    __device__ static uint32_t pack4(float a, float b, float c, float d) {
        const uint32_t i = uint32_t(int(rintf(a))) & 0xFFu, j = uint32_t(int(rintf(b))) & 0xFFu;
        const uint32_t k = uint32_t(int(rintf(c))) & 0xFFu, l = uint32_t(int(rintf(d)));
        return i | j << 8 | k << 16 | l << 24;
    }
    __device__ static void unpack4(uint32_t w, float (&f)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = float(int8_t(w >> (8 * j)));
    }
};
struct Fp8 {
    static constexpr float kTop = 448.0f;
    __device__ static uint32_t pack4(float a, float b, float c, float d) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
        return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true));
    }
    __device__ static void unpack4(uint32_t w, float (&f)[4]) {
        const f32x2 l = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), false), h = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), true);
        f[0] = l.x, f[1] = l.y, f[2] = h.x, f[3] = h.y;
    }
};

// kN elements of a tensor, as they lie in memory.  top(): the largest of their
// bits without the signs, as fp32 bits: for NaN over infinity over numbers.
template <typename Fmt, int kN>
struct Run16 {
    using S = uint16_t;
    static constexpr int kAccesses = kN / 8;
    u32x4 v[kAccesses];
    __device__ void load(const S* p) {
#pragma unroll
        for (int k = 0; k < kAccesses; ++k) v[k] = reinterpret_cast<const u32x4*>(p)[k];
    }
    __device__ void load(const S* p, uint32_t n) {
#pragma unroll
        for (int j = 0; j < kN / 2; ++j) {
            const uint32_t lo = uint32_t(2 * j) < n ? p[2 * j] : 0, hi = uint32_t(2 * j + 1) < n ? p[2 * j + 1] : 0;
            v[j / 4][j % 4] = lo | hi << 16;
        }
    }
    __device__ float get(int j) const {
        const uint32_t w = v[j / 8][j % 8 / 2];
        return j % 2 ? Fmt::hi(w) : Fmt::lo(w);
    }
    __device__ uint32_t top() const {
        uint32_t lo = 0, hi = 0;
#pragma unroll
        for (int j = 0; j < kN / 2; ++j) {
            const uint32_t w = v[j / 4][j % 4];
            lo = max(lo, w & 0x7FFFu);
            hi = max(hi, w & 0x7FFF0000u);
        }
        return __float_as_uint(Fmt::lo(max(lo, hi >> 16)));
    }
    __device__ void set(int j, float a, float b) { v[j / 8][j % 8 / 2] = Fmt::pack(a, b); }   // elements j, j + 1
    __device__ void store(S* p) const {
#pragma unroll
        for (int k = 0; k < kAccesses; ++k) reinterpret_cast<u32x4*>(p)[k] = v[k];
    }
    __device__ void store(S* p, uint32_t n) const {
#pragma unroll
        for (int j = 0; j < kN; ++j)
            if (uint32_t(j) < n) p[j] = uint16_t(v[j / 8][j % 8 / 2] >> (j % 2 * 16));
    }
};
template <int kN>
struct Run32 {
    using S = float;
    f32x4 v[kN / 4];
    __device__ void load(const S* p) {
#pragma unroll
        for (int k = 0; k < kN / 4; ++k) v[k] = reinterpret_cast<const f32x4*>(p)[k];
    }
    __device__ void load(const S* p, uint32_t n) {
#pragma unroll
        for (int j = 0; j < kN; ++j) v[j / 4][j % 4] = uint32_t(j) < n ? p[j] : 0.0f;
    }
    __device__ float get(int j) const { return v[j / 4][j % 4]; }
    __device__ uint32_t top() const {
        uint32_t t = 0;
#pragma unroll
        for (int j = 0; j < kN; ++j) t = max(t, __float_as_uint(v[j / 4][j % 4]) & 0x7FFFFFFFu);
        return t;
    }
    __device__ void set(int j, float a, float b) { v[j / 4][j % 4] = a, v[j / 4][j % 4 + 1] = b; }
    __device__ void store(S* p) const {
#pragma unroll
        for (int k = 0; k < kN / 4; ++k) reinterpret_cast<f32x4*>(p)[k] = v[k];
    }
    __device__ void store(S* p, uint32_t n) const {
#pragma unroll
        for (int j = 0; j < kN; ++j)
            if (uint32_t(j) < n) p[j] = v[j / 4][j % 4];
    }
};
template <typename Fmt>
struct Of16 {
    template <int kN>
    using Run = Run16<Fmt, kN>;
};
struct Of32 {
    template <int kN>
    using Run = Run32<kN>;
};

// kWide: x starts on a 16-byte boundary.  Lanes past the last element of the
// last block take part with zeros: every block has its lanes.
template <typename Run, typename Code, bool kWide>
__global__ __launch_bounds__(kThreads) void act8_pack_kernel(const typename Run::S* __restrict__ x, uint64_t n,
                                                             uint64_t blocks, u32x4* __restrict__ codes,
                                                             float* __restrict__ scales, uint64_t first) {
    constexpr int kShare = kBlock / kPack;   // lanes of a block
    const uint64_t lane = first + uint64_t(blockIdx.x) * kThreads + threadIdx.x;
    if (lane / kShare >= blocks) return;   // whole blocks of lanes
    const uint64_t i = lane * kPack;
    Run r;
    if (kWide && i + kPack <= n) r.load(x + i);
    else r.load(x + i, i < n ? (n - i < kPack ? uint32_t(n - i) : uint32_t(kPack)) : 0u);
    uint32_t t = r.top();
#pragma unroll
    for (int d = 1; d < kShare; d <<= 1) t = max(t, uint32_t(__shfl_xor(int(t), d)));
    u32x4 c = {0, 0, 0, 0};
    float scale = __builtin_nanf("");
    if (t < 0x7F800000u) {
        const float most = fminf(fmaxf(__uint_as_float(t), kLeast), kMost);
        const float inv = Code::kTop / most;
        scale = most / Code::kTop;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            c[k] = Code::pack4(r.get(4 * k) * inv, r.get(4 * k + 1) * inv, r.get(4 * k + 2) * inv, r.get(4 * k + 3) * inv);
    }
    codes[lane] = c;
    if (lane % kShare == 0) scales[lane / kShare] = scale;
}

template <typename Run, typename Code, bool kWide>
__global__ __launch_bounds__(kThreads) void act8_unpack_kernel(const u32x2* __restrict__ codes,
                                                               const float* __restrict__ scales, uint64_t n,
                                                               typename Run::S* __restrict__ x, uint64_t first) {
    const uint64_t lane = first + uint64_t(blockIdx.x) * kThreads + threadIdx.x;
    const uint64_t i = lane * kUnpack;
    if (i >= n) return;
    const u32x2 c = codes[lane];
    const float scale = scales[lane / (kBlock / kUnpack)];
    Run r;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        float f[4];
        Code::unpack4(c[k], f);
        r.set(4 * k, f[0] * scale, f[1] * scale);
        r.set(4 * k + 2, f[2] * scale, f[3] * scale);
    }
    if (kWide && i + kUnpack <= n) r.store(x + i);
    else r.store(x + i, n - i < kUnpack ? uint32_t(n - i) : uint32_t(kUnpack));
}

// launch(first, workgroups) in as many launches as `lanes` need.
template <typename Launch>
int in_launches(uint64_t lanes, Launch launch) {
    for (uint64_t first = 0; first < lanes; first += kMaxLanes) {
        const uint64_t some = lanes - first < kMaxLanes ? lanes - first : kMaxLanes;
        launch(first, uint32_t((some + kThreads - 1) / kThreads));
        const int e = status();
        if (e != SF_OK) return e;
    }
    return SF_OK;
}

template <typename Of, typename Code>
int pack(const void* x, uint64_t n, void* packed, hipStream_t st) {
    using Run = typename Of::template Run<kPack>;
    const uint64_t blocks = (n + kBlock - 1) / kBlock;
    const auto kernel = misaligned(x, 16) ? act8_pack_kernel<Run, Code, false> : act8_pack_kernel<Run, Code, true>;
    return in_launches(blocks * (kBlock / kPack), [&](uint64_t first, uint32_t groups) {
        hipLaunchKernelGGL(kernel, dim3(groups), dim3(kThreads), 0, st, static_cast<const typename Run::S*>(x), n, blocks,
                           static_cast<u32x4*>(packed),
                           reinterpret_cast<float*>(static_cast<char*>(packed) + blocks * kBlock), first);
    });
}

template <typename Of, typename Code>
int unpack(const void* packed, uint64_t n, void* x, hipStream_t st) {
    using Run = typename Of::template Run<kUnpack>;
    const uint64_t blocks = (n + kBlock - 1) / kBlock;
    const auto kernel = misaligned(x, 16) ? act8_unpack_kernel<Run, Code, false> : act8_unpack_kernel<Run, Code, true>;
    return in_launches((n + kUnpack - 1) / kUnpack, [&](uint64_t first, uint32_t groups) {
        hipLaunchKernelGGL(kernel, dim3(groups), dim3(kThreads), 0, st, static_cast<const u32x2*>(packed),
                           reinterpret_cast<const float*>(static_cast<const char*>(packed) + blocks * kBlock), n,
                           static_cast<typename Run::S*>(x), first);
    });
}

int check(const void* x, int dtype, size_t n, const void* packed, int format) {
    if (x == nullptr || packed == nullptr || n > (size_t(1) << 62)) return SF_EINVAL;
    if (format != SF_ACT8_INT8 && format != SF_ACT8_FP8) return SF_EINVAL;
    if (dtype != SF_DTYPE_F32 && dtype != SF_DTYPE_BF16 && dtype != SF_DTYPE_F16) return SF_EDTYPE;
    if (misaligned(x, dtype == SF_DTYPE_F32 ? 4 : 2)) return SF_EINVAL;
    if (misaligned(packed, 16)) return SF_EALIGN;
    const uintptr_t a = reinterpret_cast<uintptr_t>(x), b = reinterpret_cast<uintptr_t>(packed);
    const uintptr_t bytes = n * (dtype == SF_DTYPE_F32 ? 4 : 2), held = (n + kBlock - 1) / kBlock * SF_ACT8_BLOCK_BYTES;
    return a < b + held && b < a + bytes ? SF_EOVERLAP : SF_OK;
}

}  // namespace

extern "C" {

int sf_act8_pack(const void* x, int dtype, size_t n, void* packed, int format, sf_stream_t stream) {
    if (n == 0) return SF_OK;
    const int e = check(x, dtype, n, packed, format);
    if (e != SF_OK) return e;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const bool i8 = format == SF_ACT8_INT8;
    if (dtype == SF_DTYPE_BF16) return i8 ? pack<Of16<Bf16>, Int8>(x, n, packed, st) : pack<Of16<Bf16>, Fp8>(x, n, packed, st);
    if (dtype == SF_DTYPE_F16) return i8 ? pack<Of16<F16>, Int8>(x, n, packed, st) : pack<Of16<F16>, Fp8>(x, n, packed, st);
    return i8 ? pack<Of32, Int8>(x, n, packed, st) : pack<Of32, Fp8>(x, n, packed, st);
}

int sf_act8_unpack(const void* packed, int format, size_t n, void* x, int dtype, sf_stream_t stream) {
    if (n == 0) return SF_OK;
    const int e = check(x, dtype, n, packed, format);
    if (e != SF_OK) return e;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const bool i8 = format == SF_ACT8_INT8;
    if (dtype == SF_DTYPE_BF16) return i8 ? unpack<Of16<Bf16>, Int8>(packed, n, x, st) : unpack<Of16<Bf16>, Fp8>(packed, n, x, st);
    if (dtype == SF_DTYPE_F16) return i8 ? unpack<Of16<F16>, Int8>(packed, n, x, st) : unpack<Of16<F16>, Fp8>(packed, n, x, st);
    return i8 ? unpack<Of32, Int8>(packed, n, x, st) : unpack<Of32, Fp8>(packed, n, x, st);
}

}  // extern "C"
