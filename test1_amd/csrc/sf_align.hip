// Losses over token log-probabilities for MI355X (gfx950): the preference loss
// of paired sequences and the clipped policy loss with a KL term.
//
// Both read every token once and write its gradient once.  As separate
// elementwise and reduction operations, forward and backward, they are some 30
// to 60 launches; here they are two or three, and the host's time for a forward
// and a backward, 50 to 65 us with autograd's, is what bounds a call.  On the
// device, parts | join | gradient, us: preference, 128 x 8191 tokens 4.2 | 4.7 |
// 3.5, 9.4 MB and 5.2 MB; policy, 256 x 8191 with every input 11.3 | 4.0 | 4.9, 44
// MB, 3.9 TB/s, and 17 MB.  The sums are taken in fp32 by each lane over its few tokens
// and in fp64 from there on, in an order fixed by the shape alone: no atomics.
// Masked tokens are selected away before any arithmetic, so NaN and infinities
// there reach neither a sum nor a gradient.
//
// C ABI: include/slidefsdp.h.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/slidefsdp.h"
#include "sf_common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kSoloThreads = 1024;

// A [rows, cols] array of a call: its first element and elements from row to row.
template <typename T>
struct Rows {
    const T* p;
    uint64_t ld;
    __device__ const T* row(uint64_t r) const { return p + r * ld; }
};

// The sum over groups of kN neighbouring lanes, in every one of them.
template <int kN>
__device__ __forceinline__ double lane_sum(double x) {
#pragma unroll
    for (int d = kN / 2; d > 0; d >>= 1) x += __shfl_xor(x, d);
    return x;
}

// kN sums over a workgroup of kT lanes, in every lane.  `waves`: LDS for
// kN * kT / 64 doubles, free to use again after the caller's next barrier.
template <int kN, int kT>
__device__ __forceinline__ void block_sums(double (&x)[kN], double* waves) {
    constexpr int kWaves = kT / 64;
#pragma unroll
    for (int k = 0; k < kN; ++k) x[k] = lane_sum<64>(x[k]);
    if constexpr (kWaves > 1) {
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int k = 0; k < kN; ++k) waves[k * kWaves + (threadIdx.x >> 6)] = x[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kN; ++k) {
            x[k] = 0.0;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) x[k] += waves[k * kWaves + w];
        }
    }
}

// ---------------------------------------------------------------------
// Preference loss.  Per sequence s the sum R_s of its tokens' log ratios
// lp - ref (of the differences: the two sums apart would cancel), or their
// mean; per pair the gap D = R_chosen - R_rejected; the loss is the mean over
// the pairs of
//   sigmoid  -(1 - e) log sigmoid(b D) - e log sigmoid(-b D)
//   hinge    max(0, 1 - b D)
//   ipo      (D - 1 / (2 b))^2
// Its derivative by a token of a sequence is one number for all of them, which
// the join below writes once for each row; the backward spreads it.
// ---------------------------------------------------------------------
struct Pref {
    Rows<float> lp, ref;
    Rows<uint8_t> mask;
    uint32_t pairs, cols, splits;
    int form;
    float beta, smooth;
    bool average;
};
struct PrefOut {
    float *loss, *chosen, *rejected, *coef;
};

// The part [from, to) of one row by kN neighbouring lanes: the sum of its log
// ratios and the number of its tokens, in each of them.
template <int kN>
__device__ __forceinline__ void ratio_sum(const Pref& a, uint64_t row, uint32_t from, uint32_t to, uint32_t lane,
                                          double& sum, double& count) {
    const float *lp = a.lp.row(row), *ref = a.ref.row(row);
    const uint8_t* mask = a.mask.row(row);
    constexpr int kU = 4;   // tokens of a lane with loads in flight together
    uint32_t n = 0;
    double total = 0.0;
    for (uint32_t t = from + lane; t < to; t += kN * kU) {
        float d[kU], s = 0.0f;
        bool m[kU];
#pragma unroll
        for (int k = 0; k < kU; ++k) {
            const uint32_t u = t + k * kN;
            const bool in = u < to;
            m[k] = in && mask[in ? u : t] != 0;
            d[k] = lp[in ? u : t] - ref[in ? u : t];
        }
#pragma unroll
        for (int k = 0; k < kU; ++k) {
            s += m[k] ? d[k] : 0.0f;
            n += m[k];
        }
        total += double(s);
    }
    sum = lane_sum<kN>(total);
    count = lane_sum<kN>(double(n));
}

// log(1 + exp(-x)) for any x: -log sigmoid(x).
__device__ __forceinline__ double softplus_neg(double x) { return fmax(-x, 0.0) + log1p(exp(-fabs(x))); }

// The pairs' losses from the rows' sums, by one workgroup, kN lanes to a pair.
template <int kN>
__device__ __forceinline__ void pref_join(const Pref& a, const PrefOut& o, const double2* parts, double* waves) {
    double loss[1] = {0.0};
    const double beta = a.beta, e = a.smooth;
    const uint32_t lane = threadIdx.x % kN;
    for (uint32_t p = threadIdx.x / kN; p < a.pairs; p += kSoloThreads / kN) {
        double r[2], scale[2];
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const double2* row = parts + (p + w * uint64_t(a.pairs)) * a.splits;
            double sum = 0.0, count = 0.0;
            for (uint32_t k = lane; k < a.splits; k += kN) sum += row[k].x, count += row[k].y;
            sum = lane_sum<kN>(sum);
            count = lane_sum<kN>(count);
            scale[w] = a.average ? 1.0 / fmax(count, 1.0) : 1.0;
            r[w] = sum * scale[w];
        }
        if (lane != 0) continue;
        const double gap = r[0] - r[1], x = beta * gap;
        double term, slope;   // and its derivative by the gap
        if (a.form == SF_PREF_SIGMOID) {
            // a part that weighs nothing stays out, were it infinite
            term = (e < 1.0 ? (1.0 - e) * softplus_neg(x) : 0.0) + (e > 0.0 ? e * softplus_neg(-x) : 0.0);
            slope = beta * (e / (1.0 + exp(-x)) - (1.0 - e) / (1.0 + exp(x)));
        } else if (a.form == SF_PREF_HINGE) {
            // a NaN gap stays one; at the corner the slope is the flat side's
            term = x >= 1.0 ? 0.0 : 1.0 - x;
            slope = x >= 1.0 ? 0.0 : x != x ? x : -beta;
        } else {
            const double off = gap - 0.5 / beta;
            term = off * off;
            slope = 2.0 * off;
        }
        loss[0] += term;
        o.chosen[p] = float(beta * r[0]);
        o.rejected[p] = float(beta * r[1]);
        if (o.coef != nullptr) {
            o.coef[p] = float(slope * scale[0] / a.pairs);
            o.coef[uint64_t(a.pairs) + p] = float(-slope * scale[1] / a.pairs);
        }
    }
    block_sums<1, kSoloThreads>(loss, waves);
    if (threadIdx.x == 0) *o.loss = float(loss[0] / a.pairs);
}

// A few short sequences: one workgroup, a wave to each row in turn.
__global__ __launch_bounds__(kSoloThreads) void pref_solo_kernel(Pref a, PrefOut o, double2* __restrict__ parts) {
    __shared__ double waves[kSoloThreads / 64];
    for (uint32_t r = threadIdx.x >> 6; r < 2 * a.pairs; r += kSoloThreads / 64) {
        double s, n;
        ratio_sum<64>(a, r, 0, a.cols, threadIdx.x & 63, s, n);
        if ((threadIdx.x & 63) == 0) parts[r] = double2{s, n};
    }
    __syncthreads();
    pref_join<1>(a, o, parts, waves);
}

// A row's parts by a workgroup each.
__global__ __launch_bounds__(kThreads) void pref_parts_kernel(Pref a, uint32_t per, uint64_t first,
                                                              double2* __restrict__ parts) {
    __shared__ double waves[2 * kThreads / 64];
    const uint64_t b = first + blockIdx.x;
    const uint64_t row = b / a.splits;
    const uint32_t from = uint32_t(b % a.splits) * per, to = min(from + per, a.cols);
    double x[2];
    const uint32_t wave = threadIdx.x >> 6, each = per / (kThreads / 64);   // a multiple of 64 tokens to each wave
    ratio_sum<64>(a, row, min(from + wave * each, to), min(from + (wave + 1) * each, to), threadIdx.x & 63, x[0], x[1]);
    if ((threadIdx.x & 63) == 0) waves[wave] = x[0], waves[kThreads / 64 + wave] = x[1];
    __syncthreads();
    if (threadIdx.x == 0) {
        double s = 0.0, n = 0.0;
        for (int w = 0; w < kThreads / 64; ++w) s += waves[w], n += waves[kThreads / 64 + w];
        parts[b] = double2{s, n};
    }
}

template <int kN>
__global__ __launch_bounds__(kSoloThreads) void pref_join_kernel(Pref a, PrefOut o, const double2* __restrict__ parts) {
    __shared__ double waves[kSoloThreads / 64];
    pref_join<kN>(a, o, parts, waves);
}

// ---------------------------------------------------------------------
// Policy loss.  With d = lp - old, q = ref - lp and advantage A, a token's
// term is
//   -min(exp(d) A, clip(exp(d), 1 - low, 1 + high) A) + k (exp(q) - 1 - q),
// its derivative by lp
//   -[not clipped] exp(d) A - k (exp(q) - 1).
// Whether a token is clipped is decided on d itself, against log(1 - low) and
// log(1 + high): no rounding of the exponential turns it.
// The loss is the mean over the mask's tokens, or over the sequences that have
// any of their own means.
// ---------------------------------------------------------------------
struct Policy {
    Rows<float> lp, old, ref, adv;   // ref.p may be null
    Rows<uint8_t> mask;
    uint32_t rows, cols, splits;
    uint32_t adv_step;               // 1: an advantage for each token, 0: for each row
    float log_low, log_high, kl_coef;
    bool sequences;
};
struct PolicyOut {
    float *loss, *kl, *clipped;
    float* slope;    // [rows, cols] derivative of each token's term, or null
    float* weight;   // [rows] what its tokens weigh in the loss
};
constexpr int kSums = 4;   // terms, KL, clipped tokens, tokens
struct Sums {
    double x[kSums];
};

// exp(q) - 1 - q.  Near 0 its leading terms cancel: a series there (the first
// term left out, q^10 / 11!, is below 2^-24 of the result for |q| <= 1/2).
__device__ __forceinline__ float kl_term(float q, float em1) {
    if (fabsf(q) > 0.5f) return em1 - q;
    float s = 1.0f / 3628800.0f;
    s = fmaf(s, q, 1.0f / 362880.0f);
    s = fmaf(s, q, 1.0f / 40320.0f);
    s = fmaf(s, q, 1.0f / 5040.0f);
    s = fmaf(s, q, 1.0f / 720.0f);
    s = fmaf(s, q, 1.0f / 120.0f);
    s = fmaf(s, q, 1.0f / 24.0f);
    s = fmaf(s, q, 1.0f / 6.0f);
    s = fmaf(s, q, 0.5f);
    return s * q * q;
}

// The part [from, to) of one row by a wave: its four sums, in every lane.
__device__ __forceinline__ Sums policy_sums(const Policy& a, const PolicyOut& o, uint64_t row, uint32_t from,
                                            uint32_t to, uint32_t lane) {
    const float *lp = a.lp.row(row), *old = a.old.row(row), *adv = a.adv.row(row);
    const float* ref = a.ref.p != nullptr ? a.ref.row(row) : lp;
    const uint8_t* mask = a.mask.row(row);
    float* slope = o.slope != nullptr ? o.slope + row * a.cols : nullptr;
    constexpr int kU = 4;
    double term = 0.0, kl = 0.0;
    uint32_t clipped = 0, tokens = 0;
    for (uint32_t t = from + lane; t < to; t += 64 * kU) {
        float l[kU], d[kU], q[kU], ad[kU];
        bool m[kU];
#pragma unroll
        for (int k = 0; k < kU; ++k) {
            const uint32_t u = t + k * 64 < to ? t + k * 64 : t;
            m[k] = mask[u] != 0;
            l[k] = lp[u];
            d[k] = old[u];
            q[k] = ref[u];
            ad[k] = adv[u * a.adv_step];
        }
        float s = 0.0f, z = 0.0f;
#pragma unroll
        for (int k = 0; k < kU; ++k) {
            if (t + k * 64 >= to) break;
            float g = 0.0f;
            if (m[k]) {
                const float dd = l[k] - d[k], qq = q[k] - l[k];
                const bool clip = ad[k] > 0.0f ? dd > a.log_high : ad[k] < 0.0f && dd < a.log_low;
                const float ra = expf(clip ? (ad[k] > 0.0f ? a.log_high : a.log_low) : dd) * ad[k];
                float x = -ra;
                g = clip ? 0.0f : -ra;
                if (a.ref.p != nullptr) {
                    const float em1 = expm1f(qq), y = kl_term(qq, em1);
                    x = fmaf(a.kl_coef, y, x);
                    g = fmaf(-a.kl_coef, em1, g);
                    z += y;
                }
                s += x;
                clipped += clip;
                tokens += 1;
            }
            if (slope != nullptr) slope[t + k * 64] = g;
        }
        term += double(s);
        kl += double(z);
    }
    return {{lane_sum<64>(term), lane_sum<64>(kl), lane_sum<64>(double(clipped)), lane_sum<64>(double(tokens))}};
}

// The loss from the rows' sums, by one workgroup, kN lanes to a row.
template <int kN>
__device__ __forceinline__ void policy_join(const Policy& a, const PolicyOut& o, const Sums* parts, double* waves) {
    double total[kSums] = {0.0, 0.0, 0.0, 0.0};
    const uint32_t lane = threadIdx.x % kN;
    for (uint32_t r = threadIdx.x / kN; r < a.rows; r += kSoloThreads / kN) {
        const Sums* row = parts + uint64_t(r) * a.splits;
        double x[kSums] = {0.0, 0.0, 0.0, 0.0};
        for (uint32_t k = lane; k < a.splits; k += kN)
#pragma unroll
            for (int j = 0; j < kSums; ++j) x[j] += row[k].x[j];
#pragma unroll
        for (int j = 0; j < kSums; ++j) x[j] = lane_sum<kN>(x[j]);
        if (lane != 0) continue;
        if (a.sequences) {
            const double n = x[3];
            if (n > 0.0) {
#pragma unroll
                for (int j = 0; j < 3; ++j) x[j] /= n;
                x[3] = 1.0;
            }
        }
#pragma unroll
        for (int j = 0; j < kSums; ++j) total[j] += x[j];
    }
    block_sums<kSums, kSoloThreads>(total, waves);
    const double n = total[3];
    if (threadIdx.x == 0) {   // 0 / 0 where there is no token at all
        *o.loss = float(total[0] / n);
        if (o.kl != nullptr) *o.kl = float(total[1] / n);
        *o.clipped = float(total[2] / n);
    }
    if (o.weight == nullptr) return;
    for (uint32_t r = threadIdx.x / kN; r < a.rows; r += kSoloThreads / kN) {
        double own = 1.0;
        if (a.sequences) {
            own = 0.0;
            for (uint32_t k = lane; k < a.splits; k += kN) own += parts[uint64_t(r) * a.splits + k].x[3];
            own = lane_sum<kN>(own);
        }
        // a row without tokens has slopes of 0 alone
        if (lane == 0) o.weight[r] = own > 0.0 && n > 0.0 ? float(1.0 / (own * n)) : 0.0f;
    }
}

__global__ __launch_bounds__(kSoloThreads) void policy_solo_kernel(Policy a, PolicyOut o, Sums* __restrict__ parts) {
    __shared__ double waves[kSums * kSoloThreads / 64];
    for (uint32_t r = threadIdx.x >> 6; r < a.rows; r += kSoloThreads / 64) {
        const Sums s = policy_sums(a, o, r, 0, a.cols, threadIdx.x & 63);
        if ((threadIdx.x & 63) == 0) parts[r] = s;
    }
    __syncthreads();
    policy_join<1>(a, o, parts, waves);
}

__global__ __launch_bounds__(kThreads) void policy_parts_kernel(Policy a, PolicyOut o, uint32_t per, uint64_t first,
                                                                Sums* __restrict__ parts) {
    __shared__ Sums waves[kThreads / 64];
    const uint64_t b = first + blockIdx.x;
    const uint64_t row = b / a.splits;
    const uint32_t from = uint32_t(b % a.splits) * per, to = min(from + per, a.cols);
    const uint32_t wave = threadIdx.x >> 6, each = per / (kThreads / 64);
    const Sums s = policy_sums(a, o, row, min(from + wave * each, to), min(from + (wave + 1) * each, to), threadIdx.x & 63);
    if ((threadIdx.x & 63) == 0) waves[wave] = s;
    __syncthreads();
    if (threadIdx.x < kSums) {
        double t = 0.0;
        for (int w = 0; w < kThreads / 64; ++w) t += waves[w].x[threadIdx.x];
        parts[b].x[threadIdx.x] = t;
    }
}

template <int kN>
__global__ __launch_bounds__(kSoloThreads) void policy_join_kernel(Policy a, PolicyOut o, const Sums* __restrict__ parts) {
    __shared__ double waves[kSums * kSoloThreads / 64];
    policy_join<kN>(a, o, parts, waves);
}

// ---------------------------------------------------------------------
// Gradients: the loss's own gradient is one number on the device.
// ---------------------------------------------------------------------
constexpr int kGradPer = 4;   // tokens of a lane

__global__ __launch_bounds__(kThreads) void pref_grad_kernel(const float* __restrict__ grad_loss,
                                                             const float* __restrict__ coef, Rows<uint8_t> mask,
                                                             uint32_t cols, uint32_t col_blocks, uint64_t first,
                                                             float* __restrict__ grad) {
    const uint64_t b = first + blockIdx.x, row = b / col_blocks;
    const float c = coef[row] * *grad_loss;
    const uint8_t* m = mask.row(row);
    float* g = grad + row * cols;
    const uint32_t t = uint32_t(b % col_blocks) * (kThreads * kGradPer) + threadIdx.x;
#pragma unroll
    for (int k = 0; k < kGradPer; ++k)
        if (t + k * kThreads < cols) g[t + k * kThreads] = m[t + k * kThreads] != 0 ? c : 0.0f;
}

__global__ __launch_bounds__(kThreads) void policy_grad_kernel(const float* __restrict__ grad_loss,
                                                               const float* __restrict__ weight,
                                                               const float* __restrict__ slope, uint32_t cols,
                                                               uint32_t col_blocks, uint64_t first,
                                                               float* __restrict__ grad) {
    const uint64_t b = first + blockIdx.x, row = b / col_blocks;
    const float w = weight[row] * *grad_loss;
    const float* s = slope + row * cols;
    float* g = grad + row * cols;
    const uint32_t t = uint32_t(b % col_blocks) * (kThreads * kGradPer) + threadIdx.x;
#pragma unroll
    for (int k = 0; k < kGradPer; ++k)
        if (t + k * kThreads < cols) g[t + k * kThreads] = s[t + k * kThreads] * w;
}

// Parts of a row that one lane of the join adds up; more take a wave.  Parts and
// join together, preference | policy, us, a lane against a wave for a row: 100
// rows of 10 parts 8.5 | 10.6, 17.0 | 25.0; 64 of 16 9.5 | 11.5, 13.5 | 19.9; 32
// of 32 12.1 | 13.5, 10.1 | 14.9; 2 of 512 95 | 69, 10.9 | 11.4.
constexpr uint32_t kLaneParts = 24;

constexpr uint64_t kMaxBlocks = kMaxLanes / kThreads;

// Tokens of one part: a row is divided so that there are some 1,024 parts, each
// of 1,024 tokens or more.  us, preference | policy, at this, half and twice as
// many: 256 rows of 8191 7.9 | 13.9 (2,048 tokens), 9.3 | 15.9, 8.0 | 16.5; 128
// of 8191 8.0 | 10.6 (1,024 tokens) and, twice as many, 7.1 | 10.7.
uint32_t part_tokens(uint64_t rows, uint64_t cols) {
    const uint64_t want = (1024 + rows - 1) / rows;
    uint64_t per = (cols + want - 1) / want;
    per = (per + 1023) / 1024 * 1024;
    return uint32_t(per);
}

// Whether one workgroup takes a whole call, in one launch: where each of its waves
// has 512 tokens or fewer.  us, preference | policy, in one launch and in two,
// without the host's 3 for the second: 8 x 128 4.0 | 6.6 and 5.6 | 7.4, 8 x 512
// 4.7 | 8.6 and 5.8 | 8.0, 4 x 2048 7.3 | 17.8 and 6.0 | 8.1.
bool solo(uint64_t rows, uint64_t cols) {
    constexpr uint64_t kWaves = kSoloThreads / 64;
    return (rows + kWaves - 1) / kWaves * ((cols + 255) / 256) <= 2;
}

bool sizes_bad(size_t rows, size_t cols) {
    return rows == 0 || cols == 0 || rows > (size_t(1) << 30) || cols > (size_t(1) << 30);
}

}  // namespace

extern "C" {

size_t sf_align_parts(size_t rows, size_t cols) {
    if (sizes_bad(rows, cols)) return 0;
    const uint64_t per = part_tokens(rows, cols);
    return solo(rows, cols) ? rows : rows * ((cols + per - 1) / per);
}

int sf_pref_loss(const float* logps, size_t ld, const float* ref, size_t ld_ref, const uint8_t* mask, size_t ld_mask,
                 size_t pairs, size_t cols, int form, float beta, float smoothing, int average, void* parts,
                 float* loss, float* chosen, float* rejected, float* coef, sf_stream_t stream) {
    if (logps == nullptr || ref == nullptr || mask == nullptr || parts == nullptr || loss == nullptr ||
        chosen == nullptr || rejected == nullptr)
        return SF_EINVAL;
    if (sizes_bad(2 * pairs, cols) || pairs > (size_t(1) << 29) || ld < cols || ld_ref < cols || ld_mask < cols)
        return SF_EINVAL;
    if (form != SF_PREF_SIGMOID && form != SF_PREF_HINGE && form != SF_PREF_IPO) return SF_EINVAL;
    if (!(beta > 0.0f) || !(smoothing >= 0.0f && smoothing <= 1.0f)) return SF_EINVAL;
    if (misaligned(parts, 16)) return SF_EALIGN;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const uint64_t rows = 2 * uint64_t(pairs);
    const bool one = solo(rows, cols);
    const uint32_t per = one ? uint32_t(cols) : part_tokens(rows, cols);
    Pref a = {{logps, ld}, {ref, ld_ref}, {mask, ld_mask}, uint32_t(pairs), uint32_t(cols),
              uint32_t((cols + per - 1) / per), form, beta, smoothing, average != 0};
    const PrefOut o = {loss, chosen, rejected, coef};
    double2* p = static_cast<double2*>(parts);
    if (one) {
        hipLaunchKernelGGL(pref_solo_kernel, dim3(1), dim3(kSoloThreads), 0, st, a, o, p);
        return status();
    }
    const uint64_t blocks = rows * a.splits;
    for (uint64_t first = 0; first < blocks; first += kMaxBlocks) {
        hipLaunchKernelGGL(pref_parts_kernel, dim3(uint32_t(blocks - first < kMaxBlocks ? blocks - first : kMaxBlocks)),
                           dim3(kThreads), 0, st, a, per, first, p);
        const int e = status();
        if (e != SF_OK) return e;
    }
    hipLaunchKernelGGL(a.splits > kLaneParts ? pref_join_kernel<64> : pref_join_kernel<1>, dim3(1), dim3(kSoloThreads), 0, st, a, o, p);
    return status();
}

int sf_pref_grad(const float* grad_loss, const float* coef, const uint8_t* mask, size_t ld_mask, size_t rows,
                 size_t cols, float* grad, sf_stream_t stream) {
    if (grad_loss == nullptr || coef == nullptr || mask == nullptr || grad == nullptr || sizes_bad(rows, cols) ||
        ld_mask < cols)
        return SF_EINVAL;
    const uint32_t col_blocks = uint32_t((cols + kThreads * kGradPer - 1) / (kThreads * kGradPer));
    const uint64_t blocks = uint64_t(rows) * col_blocks;
    for (uint64_t first = 0; first < blocks; first += kMaxBlocks) {
        hipLaunchKernelGGL(pref_grad_kernel, dim3(uint32_t(blocks - first < kMaxBlocks ? blocks - first : kMaxBlocks)),
                           dim3(kThreads), 0, reinterpret_cast<hipStream_t>(stream), grad_loss, coef,
                           Rows<uint8_t>{mask, ld_mask}, uint32_t(cols), col_blocks, first, grad);
        const int e = status();
        if (e != SF_OK) return e;
    }
    return SF_OK;
}

int sf_policy_loss(const float* logps, size_t ld, const float* old_logps, size_t ld_old, const float* ref,
                   size_t ld_ref, const float* advantages, size_t ld_adv, int per_token, const uint8_t* mask,
                   size_t ld_mask, size_t rows, size_t cols, float log_low, float log_high, float kl_coef,
                   int sequences, void* parts, float* loss, float* kl, float* clipped, float* slope, float* weight,
                   sf_stream_t stream) {
    if (logps == nullptr || old_logps == nullptr || advantages == nullptr || mask == nullptr || parts == nullptr ||
        loss == nullptr || clipped == nullptr || (ref != nullptr) != (kl != nullptr))
        return SF_EINVAL;
    if (sizes_bad(rows, cols) || ld < cols || ld_old < cols || (ref != nullptr && ld_ref < cols) || ld_mask < cols ||
        (per_token && ld_adv < cols))
        return SF_EINVAL;
    if (!(log_low <= 0.0f) || !(log_high >= 0.0f)) return SF_EINVAL;
    if (misaligned(parts, 16)) return SF_EALIGN;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const bool one = solo(rows, cols);
    const uint32_t per = one ? uint32_t(cols) : part_tokens(rows, cols);
    const Policy a = {{logps, ld}, {old_logps, ld_old}, {ref, ld_ref}, {advantages, ld_adv}, {mask, ld_mask},
                      uint32_t(rows), uint32_t(cols), uint32_t((cols + per - 1) / per), per_token ? 1u : 0u,
                      log_low, log_high, kl_coef, sequences != 0};
    const PolicyOut o = {loss, kl, clipped, slope, weight};
    Sums* p = static_cast<Sums*>(parts);
    if (one) {
        hipLaunchKernelGGL(policy_solo_kernel, dim3(1), dim3(kSoloThreads), 0, st, a, o, p);
        return status();
    }
    const uint64_t blocks = uint64_t(rows) * a.splits;
    for (uint64_t first = 0; first < blocks; first += kMaxBlocks) {
        hipLaunchKernelGGL(policy_parts_kernel, dim3(uint32_t(blocks - first < kMaxBlocks ? blocks - first : kMaxBlocks)),
                           dim3(kThreads), 0, st, a, o, per, first, p);
        const int e = status();
        if (e != SF_OK) return e;
    }
    hipLaunchKernelGGL(a.splits > kLaneParts ? policy_join_kernel<64> : policy_join_kernel<1>, dim3(1), dim3(kSoloThreads), 0, st, a, o, p);
    return status();
}

int sf_policy_grad(const float* grad_loss, const float* weight, const float* slope, size_t rows, size_t cols,
                   float* grad, sf_stream_t stream) {
    if (grad_loss == nullptr || weight == nullptr || slope == nullptr || grad == nullptr || sizes_bad(rows, cols))
        return SF_EINVAL;
    const uint32_t col_blocks = uint32_t((cols + kThreads * kGradPer - 1) / (kThreads * kGradPer));
    const uint64_t blocks = uint64_t(rows) * col_blocks;
    for (uint64_t first = 0; first < blocks; first += kMaxBlocks) {
        hipLaunchKernelGGL(policy_grad_kernel, dim3(uint32_t(blocks - first < kMaxBlocks ? blocks - first : kMaxBlocks)),
                           dim3(kThreads), 0, reinterpret_cast<hipStream_t>(stream), grad_loss, weight, slope,
                           uint32_t(cols), col_blocks, first, grad);
        const int e = status();
        if (e != SF_OK) return e;
    }
    return SF_OK;
}

}  // extern "C"
