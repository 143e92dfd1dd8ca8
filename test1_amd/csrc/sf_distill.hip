// Distillation under the output unit, and the gradient of its logits, for MI355X
// (gfx950): the divergence of p = softmax(z), z = scale * hidden weight^T, from a
// teacher that leaves log-probabilities of a few words for each token.
//
// With q_k the teacher's probabilities of its words and all other words as one
// outcome, q_r = 1 - sum q_k and p_r the student's mass outside them:
//
//   forward  L = sum_b q_b (log q_b - log p_b)    v_b = Q p_b - q_b, Q = sum q_b
//   reverse  L = sum_b p_b (log p_b - log q_b)    v_b = p_b (log p_b - log q_b - L)
//
// v_k is the derivative by a named word's logit; the others share v_r by their
// softmax among themselves.  So a token needs its few words' logits exactly and of
// all others a maximum and a sum alone: logps_tiles_kernel picks the words out of a
// tile before it takes those, and log p_r is a logarithm of that sum, where 1 -
// sum p_k would have left nothing of a small rest.
//
// The gradients' products are those of the log-probabilities.  Their operand D is the
// derivative itself, upstream gradient and all, over the largest of the call, c, which
// leaves in fp32 before the results are rounded: one rounding, the hidden rows as they
// are.  Over c: where a few tokens lead, their elements are the largest of their binade,
// whose rounding is the least.  (Rows of D over their own largest and hidden rows times that,
// as the log-probabilities have it, were a rounding more in the weight gradient where no
// element of D is exact: 2.8e-3 of relative error, two roundings being 2.4e-3.)
//
// A token's few terms, q, p and L, are in 64 bits: L is a small difference of them.  The
// logits of its likely words are summed again in 64 bits: in fp32 a logit of 14 is off by
// 1e-6, as much as all else in L.
//
// C ABI: include/slidefsdp.h.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/slidefsdp.h"
#include "sf_common.h"
#include "sf_tiles.h"

namespace {

constexpr uint32_t kMost = SF_TOP_MOST;
constexpr double kLn2d = 0.69314718055994530941723;
constexpr double kLog2ed = 1.4426950408889634073599;
constexpr double kLeastRest = 0x1p-24;   // of q_r, where it is divided by: what fp32 log-probabilities tell from 0

enum Status : uint8_t { kNone, kTaught, kBad };

// ---------------------------------------------------------------------
// Each token's words by rising index, with its teacher's log-probabilities, and where
// those of each tile begin.  A wave takes a token, two words a lane, and ranks them by
// counting: 128 comparisons a lane at most, where a sort would be 28 steps with a wait
// each.  4092 tokens of 64 words, 502 tiles, 19 us; 8190 of 32 23; 126 4.4.
// ---------------------------------------------------------------------
struct Lists {
    const int64_t* ids;     // ld_ids
    const float* logps;     // ld_logps; -inf: no word
    uint64_t ld_ids, ld_logps;
    const uint8_t* mask;    // or null
    uint32_t rows, k, vocab, spans, width;   // spans of width words
    int32_t* words;         // [rows, k]
    float* teacher;         // [rows, k]
    uint8_t* starts;        // [rows, spans + 1]
    uint8_t* status;        // [rows]
};
constexpr int kListRows = 4;
__global__ __launch_bounds__(kListRows * 64) void distill_lists_kernel(const Lists a) {
    __shared__ int32_t ids[kListRows][kMost], sorted[kListRows][kMost];
    constexpr int32_t kAbsent = 0x7FFFFFFF;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t row = blockIdx.x * kListRows + wave;
    if (row >= a.rows) return;   // a whole wave; no barrier of the workgroup follows
    const bool masked = a.mask != nullptr && a.mask[row] == 0;
    int32_t id[2];
    float t[2];
    bool bad = false;
    uint32_t n = 0;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const uint32_t i = e * 64 + lane;
        id[e] = kAbsent;
        t[e] = -__builtin_inff();
        if (!masked && i < a.k) t[e] = a.logps[row * a.ld_logps + i];
        const bool there = t[e] != -__builtin_inff();
        if (there) {
            const int64_t w = a.ids[row * a.ld_ids + i];
            const bool inside = w >= 0 && w < int64_t(a.vocab);
            bad |= !inside;
            id[e] = inside ? int32_t(w) : kAbsent - 1;
        }
        ids[wave][i] = id[e];
        n += __popcll(__ballot(there));
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    uint32_t rank[2] = {0, 0};
    for (uint32_t i = 0; i < a.k; ++i) {
        const int32_t other = ids[wave][i];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const bool same = other == id[e] && i != e * 64 + lane;
            rank[e] += other < id[e] || (same && i < e * 64 + lane);
            bad |= same && id[e] != kAbsent;
        }
    }
    bad = __ballot(bad) != 0;
    const Status status = masked || n == 0 ? kNone : bad ? kBad : kTaught;
    if (status != kTaught) n = 0;
#pragma unroll
    for (int e = 0; e < 2; ++e)
        if (n > 0 && id[e] != kAbsent) {
            sorted[wave][rank[e]] = id[e];
            a.words[uint64_t(row) * a.k + rank[e]] = id[e];
            a.teacher[uint64_t(row) * a.k + rank[e]] = t[e];
        }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (uint32_t s = lane; s <= a.spans; s += 64) {   // the first word from s * width on
        uint32_t lo = 0, hi = n;
        const uint64_t from = s < a.spans ? uint64_t(s) * a.width : a.vocab;
        while (lo < hi) {
            const uint32_t mid = (lo + hi) / 2;
            if (uint64_t(sorted[wave][mid]) < from) lo = mid + 1;
            else hi = mid;
        }
        a.starts[uint64_t(row) * (a.spans + 1) + s] = uint8_t(lo);
    }
    if (lane == 0) a.status[row] = status;
}

struct Taught {
    const uint8_t* status;
    __device__ bool operator()(uint32_t i) const { return status[i] == kTaught; }
};

// ---------------------------------------------------------------------
// fp32 logits that a library product has left, a row a workgroup: the words picked out,
// -inf in their place, the others' maximum and sum as one part.  fp32 calls and rows that the
// tiles cannot take; next to the library product bound by its bytes.
// ---------------------------------------------------------------------
constexpr int kRowLanes = 256;
__global__ __launch_bounds__(kRowLanes) void distill_rows_kernel(float* logits, uint64_t ld, uint32_t vocab,
                                                                 const int32_t* __restrict__ words,
                                                                 const uint8_t* __restrict__ starts, uint32_t k,
                                                                 float scale2, float2* __restrict__ parts,
                                                                 float* __restrict__ picked) {
    __shared__ float waves[kRowLanes / 64];
    const uint64_t row = blockIdx.x;
    float* x = logits + row * ld;
    const uint32_t n = starts[row * 2 + 1];
    if (threadIdx.x < n) {
        float* at = x + words[row * k + threadIdx.x];
        picked[row * k + threadIdx.x] = *at;
        *at = -__builtin_inff();
    }
    __syncthreads();
    float m = -__builtin_inff();
    for (uint32_t j = threadIdx.x; j < vocab; j += kRowLanes) m = fmaxf(m, x[j]);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(waves[0], waves[1]), fmaxf(waves[2], waves[3]));
    const float c = base(m);
    float s = 0.0f;
    for (uint32_t j = threadIdx.x; j < vocab; j += kRowLanes) s += exp2f((x[j] - c) * scale2);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) parts[row] = float2{m, (waves[0] + waves[1]) + (waves[2] + waves[3])};
}

// ---------------------------------------------------------------------
// Each token's parts and words joined: its loss, and for a backward what D is made of.
// A workgroup takes 4 tokens: first all lanes their parts, 32 neighbouring bytes of each
// tile, then a wave each their words.
// ---------------------------------------------------------------------
struct Loss {
    const float2* parts;
    uint64_t parts_row;
    uint32_t spans, rows, k, vocab;
    int whole;             // one span of all words, of operands that the tiles do not take
    const float *picked, *teacher;
    const uint8_t *starts, *status;
    double scale;
    int form;
    bool rest;
    const void *hidden, *weight;   // of the product; a row's elements side by side
    uint64_t ldh, ldw;
    const int32_t* words;
    uint32_t terms;
    float* loss;
    float* slopes;         // [rows, k] v_k / r, or null
    float* stats;          // [4, stats_row] r, the others' maximum, log2 of their sum over it, v_r / r
    uint64_t stats_row;
};
template <typename V>
__device__ __forceinline__ V wave_sum(V v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}
__device__ __forceinline__ double wave_max(double v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v = fmax(v, __shfl_xor(v, d));
    return v;
}
// One product of a token's, by its wave, in 64 bits.  What the tiles take is read 16 bytes
// at a time.
template <typename E>
__device__ __forceinline__ double product_of(const Loss& a, uint64_t token, uint64_t word) {
    const uint32_t lane = threadIdx.x & 63;
    double s = 0.0;
    if constexpr (std::is_same_v<E, float>) {
        const float *h = static_cast<const float*>(a.hidden) + token * a.ldh, *w = static_cast<const float*>(a.weight) + word * a.ldw;
        for (uint32_t i = lane; i < a.terms; i += 64) s = fma(double(h[i]), double(w[i]), s);
        return wave_sum(s);
    } else {
        const uint16_t *h = static_cast<const uint16_t*>(a.hidden) + token * a.ldh,
                       *w = static_cast<const uint16_t*>(a.weight) + word * a.ldw;
        if (a.whole == 0)
            for (uint32_t i = lane * kGroup; i < a.terms; i += 64 * kGroup) {
                const u32x4 x = *reinterpret_cast<const u32x4*>(h + i), y = *reinterpret_cast<const u32x4*>(w + i);
#pragma unroll
                for (int j = 0; j < 4; ++j)   // the products are exact in fp32
                    s += double(E::lo(x[j]) * E::lo(y[j])) + double(E::hi(x[j]) * E::hi(y[j]));
            }
        else
            for (uint32_t i = lane; i < a.terms; i += 64) s += double(E::lo(h[i]) * E::lo(w[i]));
        return wave_sum(s);
    }
}
// A wave a token: its tiles' maxima and sums joined, its words' terms two a lane.  Bound by the
// latency of the joining and of each likely word's product: 4092 tokens of 502 tiles 43 us, 8190
// of 595 88, 126 8.
constexpr double kLikely = 1.0 / 64;   // from which a word's logit is summed again
constexpr int kLossTokens = 4;
constexpr int kLossLanes = kLossTokens * 64;
template <typename E>
__global__ __launch_bounds__(kLossLanes) void distill_loss_kernel(const Loss a) {
    __shared__ Lse waves[kLossTokens][kLossTokens];
    {
        const uint32_t t = threadIdx.x % kLossTokens, token = blockIdx.x * kLossTokens + t;
        const float scale2 = float(a.scale * kLog2ed);
        Lse p = {-__builtin_inff(), 0.0f};
        const auto merge = [=](Lse p, Lse q) {
            const float m = fmaxf(p.m, q.m), c = base(m);
            return Lse{m, (p.s == 0.0f ? 0.0f : p.s * exp2f((base(p.m) - c) * scale2)) +
                              (q.s == 0.0f ? 0.0f : q.s * exp2f((base(q.m) - c) * scale2))};
        };
        if (token < a.rows && a.status[token] == kTaught)   // the others may have no parts
            for (uint32_t k = threadIdx.x / kLossTokens; k < a.spans; k += kLossLanes / kLossTokens) {
                const float2 v = a.parts[uint64_t(k) * a.parts_row + token];
                p = merge(p, Lse{v.x, v.y});
            }
#pragma unroll
        for (int d = 32; d >= kLossTokens; d >>= 1) p = merge(p, Lse{__shfl_xor(p.m, d), __shfl_xor(p.s, d)});
        if ((threadIdx.x & 63) < kLossTokens) waves[threadIdx.x >> 6][t] = p;
        __syncthreads();
        if (threadIdx.x < kLossTokens) {
#pragma unroll
            for (int w = 1; w < kLossTokens; ++w) p = merge(p, waves[w][t]);
            waves[0][t] = p;
        }
        __syncthreads();
    }
    const uint32_t lane = threadIdx.x & 63, token = blockIdx.x * kLossTokens + (threadIdx.x >> 6);
    if (token >= a.rows) return;
    const Status status = Status(a.status[token]);
    float* const r_out = a.stats + token;
    if (status != kTaught) {
        if (lane == 0) {
            a.loss[token] = status == kBad ? __builtin_nanf("") : 0.0f;
            if (a.slopes != nullptr)
                r_out[0] = a.loss[token], r_out[a.stats_row] = r_out[2 * a.stats_row] = r_out[3 * a.stats_row] = 0.0f;
        }
        return;
    }
    const Lse others = waves[0][threadIdx.x >> 6];
    const uint32_t n = a.starts[uint64_t(token) * (a.spans + 1) + a.spans];
    const bool outside = n < a.vocab;
    double z[2], t[2], q[2];
    bool mine[2];
    const double top_others = others.s == 0.0f ? -__builtin_inf() : double(base(others.m)) * a.scale * kLog2ed;
    double top = top_others;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const uint32_t i = e * 64 + lane;
        mine[e] = i < n;
        z[e] = mine[e] ? double(a.picked[uint64_t(token) * a.k + i]) * a.scale * kLog2ed : -__builtin_inf();
        t[e] = mine[e] ? double(a.teacher[uint64_t(token) * a.k + i]) : 0.0;
        q[e] = mine[e] ? exp(t[e]) : 0.0;
        top = fmax(top, z[e]);
    }
    // the student; all relative to the largest, beside which a logarithm may be nothing
    double rest_sum, sum, log_sum;
    const auto join = [&] {
        top = wave_max(top);
        rest_sum = others.s == 0.0f ? 0.0 : double(others.s) * exp2(top_others - top);
        sum = 0.0;
#pragma unroll
        for (int e = 0; e < 2; ++e) sum += mine[e] ? exp2(z[e] - top) : 0.0;
        sum = wave_sum(sum) + rest_sum;
        log_sum = log2(sum);
    };
    join();
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const bool likely = mine[e] && (q[e] >= kLikely || exp2(z[e] - top - log_sum) >= kLikely);
        for (uint64_t those = __ballot(likely); those != 0; those &= those - 1) {
            const uint32_t i = __ffsll(static_cast<unsigned long long>(those)) - 1;
            const double s = product_of<E>(a, token, a.words[uint64_t(token) * a.k + e * 64 + i]);
            if (lane == i) z[e] = s * a.scale * kLog2ed;
        }
    }
    top = top_others;
#pragma unroll
    for (int e = 0; e < 2; ++e) top = fmax(top, z[e]);
    join();
    double lp[2], p[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) lp[e] = (z[e] - top - log_sum) * kLn2d, p[e] = mine[e] ? exp(lp[e]) : 0.0;
    // of a rest far below the mass is 0, its logarithm and what it shares are not
    const double p_rest = rest_sum / sum, lp_rest = (top_others - top + log2(double(others.s)) - log_sum) * kLn2d;
    // the teacher
    double named = wave_sum(q[0] + q[1]), q_rest = 0.0;
    if (!a.rest) {
        const double l = log(named);
#pragma unroll
        for (int e = 0; e < 2; ++e) t[e] -= l, q[e] /= named;
        named = 1.0;
    } else if (outside) {
        q_rest = fmax(1.0 - named, a.form == SF_DISTILL_REVERSE ? kLeastRest : 0.0);
    }
    double each = 0.0, v[2], v_rest;
    double loss;
    if (a.form == SF_DISTILL_FORWARD) {
#pragma unroll
        for (int e = 0; e < 2; ++e) each += q[e] == 0.0 ? 0.0 : q[e] * (t[e] - lp[e]);
        loss = wave_sum(each) + (q_rest > 0.0 ? q_rest * (log(q_rest) - lp_rest) : 0.0);
        const double all = named + q_rest;
#pragma unroll
        for (int e = 0; e < 2; ++e) v[e] = all * p[e] - q[e];
        v_rest = all * p_rest - q_rest;
    } else {
        double off[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            off[e] = p[e] == 0.0 ? 0.0 : lp[e] - t[e];
            each += p[e] * off[e];
        }
        const double off_rest = p_rest == 0.0 ? 0.0 : lp_rest - log(q_rest);
        loss = wave_sum(each) + p_rest * off_rest;
#pragma unroll
        for (int e = 0; e < 2; ++e) v[e] = p[e] * (off[e] - loss);
        v_rest = p_rest * (off_rest - loss);
    }
    if (lane == 0) a.loss[token] = float(loss);
    if (a.slopes == nullptr) return;
    if (others.s == 0.0f) v_rest = 0.0;   // there is nothing to share it
    double r = fmax(wave_max(fmax(mine[0] ? fabs(v[0]) : 0.0, mine[1] ? fabs(v[1]) : 0.0)), fabs(v_rest));
    if (loss != loss) r = __builtin_nan("");
    const float r32 = float(r);
    const double by = r32 == 0.0f ? 0.0 : 1.0 / double(r32);
#pragma unroll
    for (int e = 0; e < 2; ++e)
        if (mine[e]) a.slopes[uint64_t(token) * a.k + e * 64 + lane] = float(v[e] * by);
    if (lane == 0) {
        r_out[0] = r32;
        r_out[a.stats_row] = base(others.m);
        r_out[2 * a.stats_row] = others.s == 0.0f ? 0.0f : log2f(others.s);
        r_out[3 * a.stats_row] = float(v_rest * by);
    }
}

// ---------------------------------------------------------------------
// Gradients.
struct Weights {
    const float *grad, *r;
    const uint8_t* status;
    uint64_t n;
    float scale;
    float* weight;
    float* norm;   // or null
    float unlift;  // what takes D's kLift out
    __device__ float operator()(uint64_t i) const {
        const float g = grad[i];
        return status[i] == kNone || g == 0.0f ? 0.0f : g * scale * r[i];
    }
};

// c and what the products multiply rows by: 1, or 0 where a row has no gradient.  Behind c what
// the weight gradient is multiplied by: NaN if a token has a gradient but words that are wrong,
// whose row may not be in D.  One workgroup: 4092 tokens 5 us.
constexpr int kWeightThreads = 1024;
__global__ __launch_bounds__(kWeightThreads) void distill_weight_kernel(const Weights a) {
    __shared__ float waves[kWeightThreads / 64];
    float m = 0.0f;
    bool wrong = false;
    for (uint64_t i = threadIdx.x; i < a.n; i += kWeightThreads) {
        wrong |= a.status[i] == kBad && a.grad[i] != 0.0f;
        const float w = fabsf(a(i));
        if (__builtin_isfinite(w)) m = fmaxf(m, w);
        a.weight[i] = w == 0.0f ? 0.0f : 1.0f;
    }
    if (a.norm == nullptr) return;
    wrong = __syncthreads_or(wrong);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x != 0) return;
#pragma unroll
    for (int w = 1; w < kWeightThreads / 64; ++w) m = fmaxf(m, waves[w]);
    // so that its inverse is finite too
    m = m < 0x1p-120f ? (m > 0.0f ? 0x1p-120f : 1.0f) : fminf(m, 0x1p120f);
    a.norm[0] = m * a.unlift, a.norm[1] = 1.0f, a.norm[2] = wrong ? __builtin_nanf("") : a.norm[0];
}

struct Slopes {
    const int32_t* words;
    const uint8_t* starts;
    const float* slopes;
    const float* stats;
    uint64_t stats_row;
    const uint8_t* status;
    const float* grad;
    uint32_t k, spans;
    const int32_t* order;   // of D's rows, their number behind all; or null: the tokens' own order
};
// What a row's D is: 0 whatever its hidden states hold, NaN, or computed.
enum RowOf { kZero, kNan, kComputed };
__device__ __forceinline__ RowOf row_of(const Slopes& a, uint64_t row) {
    if (a.status[row] == kNone || a.grad[row] == 0.0f || a.stats[row] == 0.0f) return kZero;
    return a.status[row] == kBad || a.stats[row] != a.stats[row] ? kNan : kComputed;
}

// D from what the product kept, in place; as logps_keep_grad_kernel, but that a token's
// own words follow over what their lane has just stored.  Bound by its bytes, 2 read and 2
// written a logit: a fifth of the rows masked, 4092 x 128256 286 us, 8190 x 152064 720, 5.5 TB/s.
constexpr int kGradThreads = 256;
constexpr int kKeepColumns = kGradThreads * kGroup * 2;
template <typename Fmt>
__global__ __launch_bounds__(kGradThreads) void distill_keep_grad_kernel(uint16_t* __restrict__ keep, uint64_t ld,
                                                                         uint32_t tokens, uint32_t col_blocks,
                                                                         uint64_t first, const float2* __restrict__ parts,
                                                                         const Slopes a, float scale,
                                                                         const float* __restrict__ norm, uint32_t cleared) {
    const uint64_t b = first + blockIdx.x, at = b / col_blocks;
    const uint32_t live = a.order != nullptr ? uint32_t(a.order[tokens]) : tokens;
    // behind the last row as many are cleared as pad the weight gradient's sum, or all that a library's product reads
    if (at >= live && at >= max((live + 63) / 64 * 64, max(cleared, 64u))) return;
    const uint64_t row = at >= live ? tokens : a.order != nullptr ? uint64_t(a.order[at]) : at;
    const uint32_t col0 = uint32_t(b % col_blocks) * kKeepColumns, col = col0 + threadIdx.x * kGroup;
    uint16_t* k = keep + at * ld;
    const RowOf kind = row < tokens ? row_of(a, row) : kZero;
    if (kind != kComputed) {
        const uint32_t w = kind == kNan ? Fmt::kNan2 : 0u;
#pragma unroll
        for (int j = 0; j < 2; ++j)
            if (col + j * kGradThreads * kGroup < ld)
                *reinterpret_cast<u32x4*>(k + col + j * kGradThreads * kGroup) = u32x4{w, w, w, w};
        return;
    }
    // the row's weight over c, of which kLift is taken out
    const float whole = a.grad[row] * scale * a.stats[row] / (norm != nullptr ? *norm : 1.0f);
    const float m = a.stats[a.stats_row + row], l = a.stats[2 * a.stats_row + row], by = a.stats[3 * a.stats_row + row] * whole;
    const uint8_t* starts = a.starts + row * (a.spans + 1);
    const uint32_t from = starts[col0 / kSpan], to = starts[min(col0 / kSpan + kKeepColumns / kSpan, a.spans)];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const uint32_t c = col + j * kGradThreads * kGroup;
        if (c >= ld) break;
        u32x4* p = reinterpret_cast<u32x4*>(k + c);
        const u32x4 v = *p;
        const float more = fmaf(base(parts[uint64_t(c / kSpan) * tokens + row].x) - m, scale * kLog2e, -l);
        u32x4 o;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            o[i] = Fmt::pack(exp2_kept<Fmt>(v[i] & 0xFFFF, more) * by, exp2_kept<Fmt>(v[i] >> 16, more) * by);
        *p = o;
        for (uint32_t i = from; i < to; ++i) {
            const uint32_t w = a.words[row * a.k + i];
            if (w - c < uint32_t(kGroup)) k[w] = uint16_t(Fmt::pack(a.slopes[row * a.k + i] * whole, 0.0f));
        }
    }
}

// Where each token's row is among D's, -1 of those without one; a lane a token.
constexpr int kPlaceThreads = 256;
__global__ __launch_bounds__(kPlaceThreads) void distill_place_kernel(const int32_t* __restrict__ order,
                                                                      const uint8_t* __restrict__ status, uint32_t rows,
                                                                      int32_t* __restrict__ place) {
    const uint32_t i = blockIdx.x * kPlaceThreads + threadIdx.x;
    if (i >= rows) return;
    if (i < uint32_t(order[rows])) place[order[i]] = int32_t(i);
    if (status[i] != kTaught) place[i] = -1;   // the others are in the order
}

// hidden_t[j, i] = hidden[order[i], j], 0 from the last row on: the weight gradient's product
// wants them along its sum.  A tile of 64 x 64 through LDS, rows of 66 elements there, so that
// a wave's reads of a column spread over the banks.  Bound by its bytes: 4092 x 4096, a fifth of
// the rows masked, 14 us, 3.8 TB/s.
constexpr int kTurn = 64;
constexpr int kTurnThreads = 256;
__global__ __launch_bounds__(kTurnThreads) void distill_hidden_kernel(const uint16_t* __restrict__ hidden, uint64_t ldh,
                                                                      uint32_t rows, uint32_t cols,
                                                                      const int32_t* __restrict__ order,
                                                                      const float* __restrict__ by,
                                                                      uint16_t* __restrict__ out, uint64_t ldt) {
    __shared__ uint32_t tile[kTurn][kTurn / 2 + 1];
    const uint32_t across = uint32_t(ldt / kTurn), row0 = blockIdx.x % across * kTurn, col0 = blockIdx.x / across * kTurn;
    const uint32_t live = uint32_t(order[rows]);
    if (row0 >= max((live + 63) / 64 * 64, 64u)) return;   // no term of the sum
    constexpr int kEach = kTurn * kTurn / kGroup / kTurnThreads;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        const uint32_t g = k * kTurnThreads + threadIdx.x, r = g / (kTurn / kGroup), c = g % (kTurn / kGroup) * kGroup;
        u32x4 v = {0, 0, 0, 0};
        if (row0 + r < live && col0 + c < cols) {
            const uint32_t from = uint32_t(order[row0 + r]);
            if (by[from] != 0.0f) v = *reinterpret_cast<const u32x4*>(hidden + from * ldh + col0 + c);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) tile[r][c / 2 + j] = v[j];
    }
    __syncthreads();
    const uint16_t* const flat = reinterpret_cast<const uint16_t*>(tile);
    constexpr uint32_t kLd = 2 * (kTurn / 2 + 1);
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        const uint32_t g = k * kTurnThreads + threadIdx.x, c = g / (kTurn / kGroup), r = g % (kTurn / kGroup) * kGroup;
        if (col0 + c >= cols) continue;
        u32x4 v;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            v[j] = uint32_t(flat[(r + 2 * j) * kLd + c]) | uint32_t(flat[(r + 2 * j + 1) * kLd + c]) << 16;
        *reinterpret_cast<u32x4*>(out + uint64_t(col0 + c) * ldt + row0 + r) = v;
    }
}

// The hidden gradient from its sum's parts: added up, times c, rounded once, into the tokens'
// rows: 0 without a gradient, NaN of a token that has one but no row in D (words that are
// wrong).  The words from `done` on, which equal parts leave over, are added here.  live: how many
// parts there are hangs on it.  Bound by its bytes: 4092 x 4096 from 6 parts 64 us, 5.6 TB/s.
constexpr int kSumThreads = 256;
template <typename Fmt>
__global__ __launch_bounds__(kSumThreads) void distill_sum_kernel(const float* __restrict__ parts, uint32_t nparts,
                                                                  uint64_t rows, uint32_t cols,
                                                                  const int32_t* __restrict__ live,
                                                                  const int32_t* __restrict__ place,
                                                                  const float* __restrict__ by,
                                                                  const float* __restrict__ norm,
                                                                  const uint16_t* __restrict__ d, uint64_t ld,
                                                                  const uint16_t* __restrict__ weight, uint64_t ldw,
                                                                  uint32_t done, uint32_t vocab,
                                                                  uint16_t* __restrict__ out) {
    const uint32_t groups = cols / kGroup;
    const uint64_t i = uint64_t(blockIdx.x) * kSumThreads + threadIdx.x, row = i / groups;
    const uint32_t col = uint32_t(i - row * groups) * kGroup;
    if (live != nullptr) nparts = parts_of_rows(uint32_t(*live), cols, (vocab + kTerms - 1) / kTerms, nparts);
    if (row >= rows) return;
    const int32_t at = place[row];
    u32x4 o = {0, 0, 0, 0};
    if (by[row] == 0.0f) {
    } else if (at < 0) {
        o = u32x4{Fmt::kNan2, Fmt::kNan2, Fmt::kNan2, Fmt::kNan2};
    } else {
        f32x4 lo = {0.0f, 0.0f, 0.0f, 0.0f}, hi = lo;
        for (uint32_t s = 0; s < nparts; ++s) {
            const f32x4* p = reinterpret_cast<const f32x4*>(parts + (s * rows + uint32_t(at)) * cols + col);
            lo += p[0], hi += p[1];
        }
        for (uint32_t w = done; w < vocab; ++w) {
            const float f = Fmt::lo(d[uint32_t(at) * ld + w]);
            const u32x4 v = *reinterpret_cast<const u32x4*>(weight + w * ldw + col);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                lo[2 * j] = fmaf(f, Fmt::lo(v[j]), lo[2 * j]), lo[2 * j + 1] = fmaf(f, Fmt::hi(v[j]), lo[2 * j + 1]);
                hi[2 * j] = fmaf(f, Fmt::lo(v[j + 2]), hi[2 * j]), hi[2 * j + 1] = fmaf(f, Fmt::hi(v[j + 2]), hi[2 * j + 1]);
            }
        }
        const float c = *norm;
        o = u32x4{Fmt::pack(lo[0] * c, lo[1] * c), Fmt::pack(lo[2] * c, lo[3] * c), Fmt::pack(hi[0] * c, hi[1] * c),
                  Fmt::pack(hi[2] * c, hi[3] * c)};
    }
    *reinterpret_cast<u32x4*>(out + row * cols + col) = o;
}

// D in fp32 of fp32 logits, in place, a row a workgroup.
__global__ __launch_bounds__(kRowLanes) void distill_grad_kernel(float* logits, uint64_t ld, uint32_t vocab, float scale2,
                                                                 const Slopes a) {
    const uint64_t row = blockIdx.x;
    float* x = logits + row * ld;
    const RowOf kind = row_of(a, row);
    const float m = a.stats[a.stats_row + row], l = a.stats[2 * a.stats_row + row], by = a.stats[3 * a.stats_row + row];
    for (uint32_t j = threadIdx.x; j < vocab; j += kRowLanes)
        x[j] = kind == kZero ? 0.0f : kind == kNan ? __builtin_nanf("") : by == 0.0f ? 0.0f : exp2f(fmaf(x[j] - m, scale2, -l)) * by;
    if (kind != kComputed) return;
    __syncthreads();
    const uint32_t n = a.starts[row * (a.spans + 1) + a.spans];
    if (threadIdx.x < n) x[a.words[row * a.k + threadIdx.x]] = a.slopes[row * a.k + threadIdx.x];
}

// ---------------------------------------------------------------------
bool sizes_bad(size_t rows, size_t vocab, int k) {
    return vocab == 0 || vocab > (size_t(1) << 30) || rows >= (size_t(1) << 31) || k < 1 || k > int(kMost);
}
uint32_t spans_of(size_t vocab, int whole) { return whole ? 1 : uint32_t((vocab + kSpan - 1) / kSpan); }

// launch(first, n) for `n` of all units at a time, as many as a launch of `lanes` each takes.
template <typename Launch>
int in_launches(uint64_t all, uint64_t lanes, Launch launch) {
    const uint64_t most = kMaxLanes / lanes;
    for (uint64_t first = 0; first < all; first += most) {
        launch(first, uint32_t(all - first < most ? all - first : most));
        const int e = status();
        if (e != SF_OK) return e;
    }
    return SF_OK;
}

}  // namespace

extern "C" {

int sf_distill_lists(const int64_t* ids, size_t ld_ids, const float* logps, size_t ld_logps, const uint8_t* mask, size_t rows,
                     int k, size_t vocab, int whole, int32_t* words, float* teacher, uint8_t* starts, uint8_t* status_,
                     sf_stream_t stream) {
    if (rows == 0) return SF_OK;
    if (ids == nullptr || logps == nullptr || words == nullptr || teacher == nullptr || starts == nullptr ||
        status_ == nullptr || sizes_bad(rows, vocab, k) || ld_ids < size_t(k) || ld_logps < size_t(k))
        return SF_EINVAL;
    const uint32_t spans = spans_of(vocab, whole);
    return in_launches(rows, 64, [&](uint64_t r, uint32_t n) {
        const Lists a = {ids + r * ld_ids, logps + r * ld_logps, ld_ids, ld_logps, mask == nullptr ? nullptr : mask + r, n,
                         uint32_t(k), uint32_t(vocab), spans, whole ? uint32_t(vocab) : uint32_t(kSpan), words + r * k,
                         teacher + r * k, starts + r * (spans + 1), status_ + r};
        hipLaunchKernelGGL(distill_lists_kernel, dim3((n + kListRows - 1) / kListRows), dim3(kListRows * 64), 0,
                           reinterpret_cast<hipStream_t>(stream), a);
    });
}

int sf_distill_tiles(const void* weight, size_t ldw, size_t vocab, const void* hidden, size_t ldh, size_t rows,
                     size_t hidden_size, const int32_t* words, const uint8_t* starts, const uint8_t* status_, int k,
                     float scale, int dtype, void* parts, float* picked, int32_t* order, void* keep, size_t ld_keep,
                     int close, sf_stream_t stream) {
    if (rows == 0) return SF_OK;
    if (weight == nullptr || hidden == nullptr || words == nullptr || starts == nullptr || status_ == nullptr ||
        parts == nullptr || picked == nullptr || sizes_bad(rows, vocab, k))
        return SF_EINVAL;
    constexpr size_t kMostLd = size_t(1) << 22;   // 32-bit byte offsets inside a tile of 256 rows
    if (hidden_size == 0 || ldw < hidden_size || ldh < hidden_size || ldw > kMostLd || ldh > kMostLd || !(scale > 0.0f))
        return SF_EINVAL;
    if (dtype != SF_DTYPE_BF16 && dtype != SF_DTYPE_F16) return SF_EDTYPE;
    const size_t spans = spans_of(vocab, 0);
    if (close && order == nullptr) return SF_EINVAL;
    if (keep != nullptr && ld_keep < spans * kSpan) return SF_EINVAL;
    if (hidden_size % kTerms != 0 || ldw % kGroup != 0 || ldh % kGroup != 0 || misaligned(weight, 16) ||
        misaligned(hidden, 16) || misaligned(parts, 8) || misaligned(keep, 16) || ld_keep % kGroup != 0)
        return SF_EALIGN;
    if (order != nullptr && uint64_t(rows) * ldh * 2 > UINT32_MAX) return SF_ETOOBIG;   // 32-bit byte offsets of all rows
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const uint64_t most = kMaxLanes / kTileKinds[0].lanes / spans * 256;   // rows of one launch, whole tiles
    if (close && rows > most) return SF_EINVAL;   // one order for all
    for (uint64_t r = 0; r < rows; r += most) {
        const uint32_t n = uint32_t(rows - r < most ? rows - r : most);
        const Tiles a = {static_cast<const uint16_t*>(weight), static_cast<const uint16_t*>(hidden) + r * ldh,
                         uint32_t(ldw), uint32_t(ldh), uint32_t(vocab), n, uint32_t(hidden_size / kTerms), nullptr,
                         order == nullptr ? nullptr : order + r, scale * kLog2e, static_cast<float2*>(parts) + r, rows,
                         nullptr, keep == nullptr ? nullptr : static_cast<uint16_t*>(keep) + r * ld_keep, ld_keep,
                         words + r * k, starts + r * (spans + 1), picked + r * k, uint32_t(k), close != 0};
        int e = SF_OK;
        if (order != nullptr) {   // its last element is the next launch's first, which is written behind this one's
            hipLaunchKernelGGL(logps_order_kernel<Taught>, dim3(1), dim3(kOrderThreads), 0, st, Taught{status_ + r}, n,
                               order + r);
            e = status();
            if (e != SF_OK) return e;
        }
        e = dtype == SF_DTYPE_BF16 ? dispatch_tiles<Bf16, true>(a, st) : dispatch_tiles<F16, true>(a, st);
        if (e != SF_OK) return e;
    }
    return SF_OK;
}

int sf_distill_rows(float* logits, size_t ld, size_t rows, size_t vocab, const int32_t* words, const uint8_t* starts, int k,
                    float scale, void* parts, float* picked, sf_stream_t stream) {
    if (rows == 0) return SF_OK;
    if (logits == nullptr || words == nullptr || starts == nullptr || parts == nullptr || picked == nullptr ||
        sizes_bad(rows, vocab, k) || ld < vocab || !(scale > 0.0f))
        return SF_EINVAL;
    if (misaligned(logits, 4) || misaligned(parts, 8)) return SF_EALIGN;
    return in_launches(rows, kRowLanes, [&](uint64_t r, uint32_t n) {
        hipLaunchKernelGGL(distill_rows_kernel, dim3(n), dim3(kRowLanes), 0, reinterpret_cast<hipStream_t>(stream),
                           logits + r * ld, uint64_t(ld), uint32_t(vocab), words + r * k, starts + r * 2, uint32_t(k),
                           scale * kLog2e, static_cast<float2*>(parts) + r, picked + r * k);
    });
}

int sf_distill_loss(const void* parts, size_t parts_row, int whole, const float* picked, const float* teacher,
                    const uint8_t* starts, const uint8_t* status_, size_t rows, int k, size_t vocab, double scale, int form,
                    int rest, const void* hidden, size_t ldh, const void* weight, size_t ldw, size_t hidden_size, int dtype,
                    const int32_t* words, float* loss, float* slopes, float* stats, size_t stats_row, sf_stream_t stream) {
    if (rows == 0) return SF_OK;
    if (parts == nullptr || picked == nullptr || teacher == nullptr || starts == nullptr || status_ == nullptr ||
        loss == nullptr || sizes_bad(rows, vocab, k) || parts_row < rows || !(scale > 0.0) ||
        (slopes != nullptr && (stats == nullptr || stats_row < rows)) || hidden == nullptr || weight == nullptr ||
        words == nullptr || hidden_size == 0 || hidden_size > (size_t(1) << 31) || ldh < hidden_size || ldw < hidden_size)
        return SF_EINVAL;
    if (dtype != SF_DTYPE_F32 && dtype != SF_DTYPE_BF16 && dtype != SF_DTYPE_F16) return SF_EDTYPE;
    if ((form != SF_DISTILL_FORWARD && form != SF_DISTILL_REVERSE) || (form == SF_DISTILL_REVERSE && !rest)) return SF_EINVAL;
    const size_t item = dtype == SF_DTYPE_F32 ? 4 : 2;
    if (misaligned(parts, 8) || misaligned(hidden, item) || misaligned(weight, item)) return SF_EALIGN;
    if (!whole && (dtype == SF_DTYPE_F32 || hidden_size % kGroup != 0 || ldh % kGroup != 0 || ldw % kGroup != 0 ||
                   misaligned(hidden, 16) || misaligned(weight, 16)))
        return SF_EALIGN;
    const uint32_t spans = spans_of(vocab, whole);
    const auto kernel = dtype == SF_DTYPE_F32    ? distill_loss_kernel<float>
                        : dtype == SF_DTYPE_BF16 ? distill_loss_kernel<Bf16>
                                                 : distill_loss_kernel<F16>;
    return in_launches(rows, 64, [&](uint64_t r, uint32_t n) {
        const Loss a = {static_cast<const float2*>(parts) + r, parts_row, spans, n, uint32_t(k), uint32_t(vocab), whole,
                        picked + r * k, teacher + r * k, starts + r * (spans + 1), status_ + r, scale, form, rest != 0,
                        static_cast<const uint8_t*>(hidden) + r * ldh * item, weight, ldh, ldw, words + r * k,
                        uint32_t(hidden_size), loss + r, slopes == nullptr ? nullptr : slopes + r * k, stats == nullptr ? nullptr : stats + r,
                        stats_row};
        hipLaunchKernelGGL(kernel, dim3((n + kLossTokens - 1) / kLossTokens), dim3(kLossLanes), 0,
                           reinterpret_cast<hipStream_t>(stream), a);
    });
}

int sf_distill_keep_grad(void* keep, size_t ld, size_t rows, size_t padded, size_t vocab, const void* parts,
                         const int32_t* words, const uint8_t* starts, const uint8_t* status_, int k, const float* slopes,
                         const float* stats, size_t stats_row, int dtype, const float* grad, float scale, const float* norm,
                         const int32_t* order, size_t cleared, sf_stream_t stream) {
    if (padded == 0) return SF_OK;
    if (keep == nullptr || parts == nullptr || words == nullptr || starts == nullptr || status_ == nullptr ||
        slopes == nullptr || stats == nullptr || stats_row < rows || sizes_bad(padded, vocab, k) || padded < rows ||
        cleared > padded || (rows > 0 && grad == nullptr) || ld < size_t(spans_of(vocab, 0)) * kSpan || ld > (size_t(1) << 31))
        return SF_EINVAL;
    if (dtype != SF_DTYPE_BF16 && dtype != SF_DTYPE_F16) return SF_EDTYPE;
    if (dtype == SF_DTYPE_F16 && norm == nullptr) return SF_EINVAL;
    if (misaligned(keep, 16) || misaligned(parts, 8) || ld % kSpan != 0) return SF_EALIGN;
    const uint32_t col_blocks = uint32_t((ld + kKeepColumns - 1) / kKeepColumns);
    const auto kernel = dtype == SF_DTYPE_BF16 ? distill_keep_grad_kernel<Bf16> : distill_keep_grad_kernel<F16>;
    const Slopes a = {words, starts, slopes, stats, stats_row, status_, grad, uint32_t(k), spans_of(vocab, 0), order};
    return in_launches(uint64_t(padded) * col_blocks, kGradThreads, [&](uint64_t first, uint32_t blocks) {
        hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kGradThreads), 0, reinterpret_cast<hipStream_t>(stream),
                           static_cast<uint16_t*>(keep), uint64_t(ld), uint32_t(rows), col_blocks, first,
                           static_cast<const float2*>(parts), a, scale, norm,
                           order == nullptr ? uint32_t(padded) : uint32_t(cleared));
    });
}

int sf_distill_weight(const float* grad, const float* stats, const uint8_t* status_, size_t rows, float scale, int dtype,
                      float* row_weight, float* norm, sf_stream_t stream) {
    if (rows == 0) return SF_OK;
    if (grad == nullptr || stats == nullptr || status_ == nullptr || row_weight == nullptr || rows >= (size_t(1) << 31))
        return SF_EINVAL;
    if (dtype != SF_DTYPE_BF16 && dtype != SF_DTYPE_F16) return SF_EDTYPE;
    const Weights a = {grad, stats, status_, rows, scale, row_weight, norm, dtype == SF_DTYPE_F16 ? 1.0f / kLift<F16> : 1.0f};
    hipLaunchKernelGGL(distill_weight_kernel, dim3(1), dim3(kWeightThreads), 0, reinterpret_cast<hipStream_t>(stream), a);
    return status();
}

int sf_distill_hidden(const void* hidden, size_t ldh, size_t rows, size_t cols, const int32_t* order, const float* row_weight,
                      void* hidden_t, size_t ldt, sf_stream_t stream) {
    if (rows == 0 || cols == 0) return SF_OK;
    if (hidden == nullptr || order == nullptr || row_weight == nullptr || hidden_t == nullptr || ldh < cols || ldt < rows ||
        ldt % kTurn != 0 || ldt - rows >= kTurn || rows >= (size_t(1) << 31) || cols > (size_t(1) << 22))
        return SF_EINVAL;
    if (misaligned(hidden, 16) || ldh % kGroup != 0 || cols % kGroup != 0 || misaligned(hidden_t, 16)) return SF_EALIGN;
    const uint64_t tiles = uint64_t(ldt / kTurn) * ((cols + kTurn - 1) / kTurn);
    if (tiles > kMaxLanes / kTurnThreads) return SF_EINVAL;
    hipLaunchKernelGGL(distill_hidden_kernel, dim3(uint32_t(tiles)), dim3(kTurnThreads), 0,
                       reinterpret_cast<hipStream_t>(stream), static_cast<const uint16_t*>(hidden), uint64_t(ldh),
                       uint32_t(rows), uint32_t(cols), order, row_weight, static_cast<uint16_t*>(hidden_t), uint64_t(ldt));
    return status();
}

int sf_distill_sum(const float* parts, int nparts, int by_live, size_t rows, size_t cols, const int32_t* order, const uint8_t* status_,
                   int32_t* place, const float* row_weight, const float* norm, const void* d, size_t ld, const void* weight,
                   size_t ldw, size_t done, size_t vocab, int dtype, void* out, sf_stream_t stream) {
    if (rows == 0 || cols == 0) return SF_OK;
    if (parts == nullptr || nparts < 1 || order == nullptr || status_ == nullptr || place == nullptr || norm == nullptr ||
        row_weight == nullptr || d == nullptr || weight == nullptr || out == nullptr || done > vocab || (by_live && (done < vocab || nparts > int(kMostLiveParts))) || ld < vocab || ldw < cols ||
        rows >= (size_t(1) << 31) || vocab > (size_t(1) << 30) || cols > (size_t(1) << 22))
        return SF_EINVAL;
    if (dtype != SF_DTYPE_BF16 && dtype != SF_DTYPE_F16) return SF_EDTYPE;
    if (cols % kGroup != 0 || ldw % kGroup != 0 || misaligned(parts, 16) || misaligned(weight, 16) || misaligned(out, 16))
        return SF_EALIGN;
    const uint64_t blocks = (uint64_t(rows) * (cols / kGroup) + kSumThreads - 1) / kSumThreads;
    if (blocks > kMaxLanes / kSumThreads) return SF_EINVAL;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(distill_place_kernel, dim3(uint32_t((rows + kPlaceThreads - 1) / kPlaceThreads)), dim3(kPlaceThreads), 0,
                       st, order, status_, uint32_t(rows), place);
    const int e = status();
    if (e != SF_OK) return e;
    const auto kernel = dtype == SF_DTYPE_BF16 ? distill_sum_kernel<Bf16> : distill_sum_kernel<F16>;
    hipLaunchKernelGGL(kernel, dim3(uint32_t(blocks)), dim3(kSumThreads), 0, st, parts, uint32_t(nparts), uint64_t(rows),
                       uint32_t(cols), by_live ? order + rows : nullptr, place, row_weight, norm, static_cast<const uint16_t*>(d), uint64_t(ld),
                       static_cast<const uint16_t*>(weight), uint64_t(ldw), uint32_t(done), uint32_t(vocab),
                       static_cast<uint16_t*>(out));
    return status();
}

int sf_distill_grad(float* logits, size_t ld, size_t rows, size_t vocab, const int32_t* words, const uint8_t* starts,
                    const uint8_t* status_, int k, float scale, const float* slopes, const float* stats, size_t stats_row,
                    const float* grad, sf_stream_t stream) {
    if (rows == 0) return SF_OK;
    if (logits == nullptr || words == nullptr || starts == nullptr || status_ == nullptr || slopes == nullptr ||
        stats == nullptr || grad == nullptr || stats_row < rows || sizes_bad(rows, vocab, k) || ld < vocab || !(scale > 0.0f))
        return SF_EINVAL;
    if (misaligned(logits, 4)) return SF_EALIGN;
    return in_launches(rows, kRowLanes, [&](uint64_t r, uint32_t n) {
        const Slopes a = {words + r * k, starts + r * 2, slopes + r * k, stats + r, stats_row, status_ + r, grad + r,
                          uint32_t(k), 1, nullptr};
        hipLaunchKernelGGL(distill_grad_kernel, dim3(n), dim3(kRowLanes), 0, reinterpret_cast<hipStream_t>(stream),
                           logits + r * ld, uint64_t(ld), uint32_t(vocab), scale * kLog2e, a);
    });
}

}  // extern "C"
