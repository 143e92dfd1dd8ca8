// Log-probabilities of given tokens under the output unit, and their
// gradient, for MI355X (gfx950).
//
// C ABI: include/slidefsdp.h.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/slidefsdp.h"
#include "sf_common.h"

namespace {

// fp32 logits that a library product has left: kT lanes per row, one pass, each
// lane with its own running maximum and sum.
template <int kT>
__global__ __launch_bounds__(kT * kRowsOf<kT>) void logps_rows_kernel(const float* __restrict__ logits, uint64_t ld,
                                                                      uint64_t rows, uint32_t vocab,
                                                                      const int64_t* __restrict__ labels,
                                                                      int64_t ignore_index, float scale,
                                                                      float* __restrict__ lse_out,
                                                                      float* __restrict__ logp_out) {
    __shared__ Lse parts[kT > 64 ? kT / 64 : 1];
    const uint32_t lane = threadIdx.x % kT;
    const uint64_t row = uint64_t(blockIdx.x) * kRowsOf<kT> + threadIdx.x / kT;
    if (kRowsOf<kT> > 1 && row >= rows) return;   // no barrier below for these
    const float* x = logits + row * ld;
    const int64_t y = labels[row];
    const RowKind kind = row_kind(y, ignore_index, vocab);
    if (kind != kValid) {
        if (lane == 0) lse_out[row] = logp_out[row] = kind == kIgnored ? 0.0f : __builtin_nanf("");
        return;
    }
    const f32x4* xv = reinterpret_cast<const f32x4*>(x);
    const uint32_t groups = vocab / 4;
    constexpr int kU = 4;
    Lse p = {-__builtin_inff(), 0.0f};
    for (uint32_t g = lane; g < groups; g += kT * kU) {
        f32x4 v[kU];
        float m = -__builtin_inff();
#pragma unroll
        for (int k = 0; k < kU; ++k) {
            const uint32_t at = g + k * kT;
            v[k] = xv[at < groups ? at : g] * scale;
            if (at >= groups) v[k] = f32x4{m, m, m, m};
        }
#pragma unroll
        for (int k = 0; k < kU; ++k) m = fmaxf(m, fmaxf(fmaxf(v[k].x, v[k].y), fmaxf(v[k].z, v[k].w)));
        m = fmaxf(m, p.m);
        const float c = base(m);
        float s = p.s == 0.0f ? 0.0f : p.s * expf(base(p.m) - c);
#pragma unroll
        for (int k = 0; k < kU; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) s += expf(v[k][j] - c);
        p = {m, s};
    }
    if (groups * 4 + lane < vocab) {   // the last elements, fewer than four
        const float f = x[groups * 4 + lane] * scale, m = fmaxf(f, p.m), c = base(m);
        p = {m, (p.s == 0.0f ? 0.0f : p.s * expf(base(p.m) - c)) + expf(f - c)};
    }
    const float lse = block_lse<kT>(p, parts);
    if (lane == 0) {
        lse_out[row] = lse;
        logp_out[row] = x[y] * scale - lse;
    }
}

// What an fp16 gradient of the logits is multiplied by: a power of two that
// brings the largest element of the gradient of the log-probabilities into [1,
// 2), since per-token gradients are of the order 1 / tokens and a probability
// times that is below fp16's range.  norm: the factor, its inverse, 1.
constexpr int kNormThreads = 1024;
__global__ __launch_bounds__(kNormThreads) void logps_norm_kernel(const float* __restrict__ grad,
                                                                  const int64_t* __restrict__ labels,
                                                                  int64_t ignore_index, uint64_t n, float scale,
                                                                  float* __restrict__ norm) {
    __shared__ float waves[kNormThreads / 64];
    float m = 0.0f;
    for (uint64_t i = threadIdx.x; i < n; i += kNormThreads) {
        const float g = fabsf(grad[i] * scale);
        if (labels[i] != ignore_index && __builtin_isfinite(g)) m = fmaxf(m, g);
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kNormThreads / 64; ++w) m = fmaxf(m, waves[w]);
        // within what both the factor and its inverse can be
        const int e = m > 0.0f ? min(max(ilogbf(m), -100), 100) : 0;
        norm[0] = ldexpf(1.0f, -e);
        norm[1] = ldexpf(1.0f, e);
        norm[2] = 1.0f;
    }
}

// Its gradient, element by element; a workgroup takes 1,024 columns of a row.
constexpr int kGradThreads = 256;
constexpr int kGradColumns = 1024;

struct Out32 {
    using S = float;
    __device__ static void store(S* p, float f) { *p = f; }
};
template <typename Fmt>
struct Out16 {
    using S = uint16_t;
    __device__ static void store(S* p, float f) { *p = uint16_t(Fmt::pack(f, 0.0f)); }
};

template <typename Out>
__global__ __launch_bounds__(kGradThreads) void logps_grad_kernel(const float* logits, uint64_t ld, uint32_t vocab,
                                                                  uint32_t col_blocks, uint64_t first,
                                                                  const int64_t* __restrict__ labels,
                                                                  int64_t ignore_index, float scale,
                                                                  const float* __restrict__ lse,
                                                                  const float* __restrict__ grad,
                                                                  const float* __restrict__ norm,
                                                                  typename Out::S* dz, uint64_t ld_dz) {
    const uint64_t b = first + blockIdx.x, row = b / col_blocks;
    const uint32_t col = uint32_t(b % col_blocks) * kGradColumns + threadIdx.x;
    const int64_t y = labels[row];
    const RowKind kind = row_kind(y, ignore_index, vocab);
    const float* x = logits + row * ld;
    typename Out::S* o = dz + row * ld_dz;
    const float l = lse[row], by = norm != nullptr ? *norm : 1.0f;
    const float g = kind == kIgnored ? 0.0f : grad[row] * scale * by;
#pragma unroll
    for (int k = 0; k < kGradColumns / kGradThreads; ++k) {
        const uint32_t j = col + k * kGradThreads;
        if (j >= vocab) break;
        float f = 0.0f;
        if (kind == kBadLabel) f = __builtin_nanf("");
        if (kind == kValid) f = g * ((int64_t(j) == y ? 1.0f : 0.0f) - expf(x[j] * scale - l));
        Out::store(o + j, f);
    }
}

template <int kT>
int launch_rows(const float* x, uint64_t ld, uint64_t rows, uint32_t vocab, const int64_t* labels, int64_t ignore,
                float scale, float* lse, float* logp, hipStream_t st) {
    constexpr uint64_t kMax = kMaxLanes / kT;
    for (uint64_t r = 0; r < rows; r += kMax) {
        const uint64_t n = rows - r < kMax ? rows - r : kMax;
        hipLaunchKernelGGL(logps_rows_kernel<kT>, dim3(uint32_t((n + kRowsOf<kT> - 1) / kRowsOf<kT>)),
                           dim3(kT * kRowsOf<kT>), 0, st, x + r * ld, ld, n, vocab, labels + r, ignore, scale, lse + r,
                           logp + r);
        const int e = status();
        if (e != SF_OK) return e;
    }
    return SF_OK;
}

template <typename Out>
int launch_grad(const float* x, uint64_t ld, uint64_t rows, uint32_t vocab, const int64_t* labels, int64_t ignore,
                float scale, const float* lse, const float* grad, const float* norm, void* dz, uint64_t ld_dz,
                hipStream_t st) {
    constexpr uint64_t kMax = kMaxLanes / kGradThreads;
    const uint32_t col_blocks = (vocab + kGradColumns - 1) / kGradColumns;
    const uint64_t blocks = rows * col_blocks;
    for (uint64_t first = 0; first < blocks; first += kMax) {
        hipLaunchKernelGGL(logps_grad_kernel<Out>, dim3(uint32_t(blocks - first < kMax ? blocks - first : kMax)),
                           dim3(kGradThreads), 0, st, x, ld, vocab, col_blocks, first, labels, ignore, scale, lse, grad,
                           norm, static_cast<typename Out::S*>(dz), ld_dz);
        const int e = status();
        if (e != SF_OK) return e;
    }
    return SF_OK;
}

bool sizes_bad(size_t rows, size_t vocab) {
    return vocab == 0 || vocab > (size_t(1) << 30) || rows >= (size_t(1) << 31);
}

}  // namespace

extern "C" {

int sf_logps_rows(const float* logits, size_t ld, size_t rows, size_t vocab, const int64_t* labels,
                  int64_t ignore_index, float scale, float* lse, float* logp, sf_stream_t stream) {
    if (rows == 0) return SF_OK;
    if (logits == nullptr || labels == nullptr || lse == nullptr || logp == nullptr) return SF_EINVAL;
    if (sizes_bad(rows, vocab) || ld < vocab) return SF_EINVAL;
    if (misaligned(logits, 16) || ld % 4 != 0) return SF_EALIGN;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const uint32_t v = uint32_t(vocab);
    if (v <= 256) return launch_rows<16>(logits, ld, rows, v, labels, ignore_index, scale, lse, logp, st);
    if (v <= 1024) return launch_rows<64>(logits, ld, rows, v, labels, ignore_index, scale, lse, logp, st);
    if (v <= 16384) return launch_rows<256>(logits, ld, rows, v, labels, ignore_index, scale, lse, logp, st);
    return launch_rows<1024>(logits, ld, rows, v, labels, ignore_index, scale, lse, logp, st);
}

int sf_logps_norm(const float* grad, const int64_t* labels, int64_t ignore_index, size_t rows, float scale, float* norm,
                  sf_stream_t stream) {
    if (norm == nullptr || (rows > 0 && (grad == nullptr || labels == nullptr))) return SF_EINVAL;
    hipLaunchKernelGGL(logps_norm_kernel, dim3(1), dim3(kNormThreads), 0, reinterpret_cast<hipStream_t>(stream), grad,
                       labels, ignore_index, uint64_t(rows), scale, norm);
    return status();
}

int sf_logps_grad(const float* logits, size_t ld, size_t rows, size_t vocab, const int64_t* labels,
                  int64_t ignore_index, float scale, const float* lse, const float* grad, const float* norm, void* dz,
                  int dtype, size_t ld_dz, sf_stream_t stream) {
    if (rows == 0) return SF_OK;
    if (logits == nullptr || labels == nullptr || lse == nullptr || grad == nullptr || dz == nullptr) return SF_EINVAL;
    if (sizes_bad(rows, vocab) || ld < vocab || ld_dz < vocab) return SF_EINVAL;
    if (dtype != SF_DTYPE_F32 && dtype != SF_DTYPE_BF16 && dtype != SF_DTYPE_F16) return SF_EDTYPE;
    const size_t item = dtype == SF_DTYPE_F32 ? 4 : 2;
    if (misaligned(dz, item)) return SF_EINVAL;
    const uintptr_t a = reinterpret_cast<uintptr_t>(logits), b = reinterpret_cast<uintptr_t>(dz);
    const uintptr_t a_end = a + ((rows - 1) * ld + vocab) * 4, b_end = b + ((rows - 1) * ld_dz + vocab) * item;
    const bool in_place = dtype == SF_DTYPE_F32 && a == b && ld == ld_dz;
    if (!in_place && a < b_end && b < a_end) return SF_EOVERLAP;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const uint32_t v = uint32_t(vocab);
    if (dtype == SF_DTYPE_BF16)
        return launch_grad<Out16<Bf16>>(logits, ld, rows, v, labels, ignore_index, scale, lse, grad, norm, dz, ld_dz, st);
    if (dtype == SF_DTYPE_F16)
        return launch_grad<Out16<F16>>(logits, ld, rows, v, labels, ignore_index, scale, lse, grad, norm, dz, ld_dz, st);
    return launch_grad<Out32>(logits, ld, rows, v, labels, ignore_index, scale, lse, grad, norm, dz, ld_dz, st);
}

}  // extern "C"
