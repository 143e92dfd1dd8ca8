// Log-probabilities of given tokens under the output unit, and the gradient
// of its logits, for MI355X (gfx950).
//
// With logits z = scale * hidden weight^T, a token's log-probability is z_y -
// log sum_j exp z_j.  16-bit operands go through logps_tiles_kernel, the
// product and the softmax's sums in one: a 256-word tile of a token's logits
// never leaves the registers, only its maximum and its sum of exponentials do
// (8 bytes for 256 logits), and the joined sums give the result.  Where a
// gradient will be wanted the exponentials themselves are kept, relative to
// their tile's maximum, 2 bytes a logit: from those a probability is off by a
// rounding of itself, from logits in 16 bits by up to 2^-8 of the logit.
// Others (fp32, hidden sizes that are no multiple of 64, unaligned rows) have
// their logits made by a library product in chunks of fp32 and read once.
//
// The gradient by the logits of token i is g_i (onehot - p).  Its operand of the
// two products is D = (onehot - p) / (1 - p_y), 1 at the label, and g_i (1 -
// p_y) multiplies a row of the hidden gradient afterwards, a hidden row before
// the weight gradient's product.  The label's element is the largest one: in D
// it is exact, where rounding g (onehot - p) to 16 bits cost as much as the
// results' own rounding (relative error of both gradients 2.4e-3 before,
// 1.7e-3 being the rounding alone).
//
// What is kept and D are at most 1, and most of a large vocabulary's elements are
// far below 2^-14, where fp16 loses bits (below 2^-25 all of them).  fp16 holds
// both times 2^14, which the fp32 factors of the results take out again: full
// precision down to 2^-28, at the cost of that product and of fewer zeros on the
// way: 4092 x 4096 x 128256 with both gradients 9.52 | 9.69 ms, 777 x 1024 x 50257
// 323 | 327 us.
//
// C ABI: include/slidefsdp.h.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/slidefsdp.h"
#include "sf_common.h"
#include "sf_tiles.h"

namespace {

constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kLeastRest = 0x1p-24f;   // of 1 - p_y, so that it can be divided by

// 1 - p of a log-probability; NaN stays NaN.
__device__ __forceinline__ float rest_of(float logp) {
    const float rest = -expm1f(logp);
    return rest < kLeastRest ? kLeastRest : rest;
}

struct HasLabel {   // inside the vocabulary
    const int64_t* labels;
    int64_t ignore_index;
    uint32_t vocab;
    __device__ bool operator()(uint32_t i) const { return row_kind(labels[i], ignore_index, vocab) == kValid; }
};

// The tiles' parts of each token joined.  A workgroup takes 4 tokens, 64 lanes
// each, so that a wave reads 32 neighbouring bytes of each tile.
constexpr int kJoinThreads = 256;
constexpr int kJoinTokens = 4;
__global__ __launch_bounds__(kJoinThreads) void logps_join_kernel(const float2* __restrict__ parts, uint32_t spans,
                                                                  uint64_t parts_row, uint32_t tokens,
                                                                  const float* __restrict__ target,
                                                                  const int64_t* __restrict__ labels,
                                                                  int64_t ignore_index, uint32_t vocab, float scale2,
                                                                  float* __restrict__ lse2, float* __restrict__ logp) {
    __shared__ Lse waves[kJoinThreads / 64][kJoinTokens];
    const uint32_t t = threadIdx.x % kJoinTokens, token = blockIdx.x * kJoinTokens + t;
    Lse p = {-__builtin_inff(), 0.0f};
    const RowKind kind = token < tokens ? row_kind(labels[token], ignore_index, vocab) : kIgnored;
    if (kind == kValid)   // the others may have no parts
        for (uint32_t k = threadIdx.x / kJoinTokens; k < spans; k += kJoinThreads / kJoinTokens) {
            const float2 v = parts[uint64_t(k) * parts_row + token];
            const float m = fmaxf(p.m, v.x), c = base(m);
            // an empty part stays empty whatever the bases are; a NaN sum stays NaN
            p.s = (p.s == 0.0f ? 0.0f : p.s * exp2f(base(p.m) - c)) + (v.y == 0.0f ? 0.0f : v.y * exp2f(base(v.x) - c));
            p.m = m;
        }
    const auto merge = [](Lse p, Lse q) {
        const float m = fmaxf(p.m, q.m), c = base(m);
        return Lse{m, (p.s == 0.0f ? 0.0f : p.s * exp2f(base(p.m) - c)) + (q.s == 0.0f ? 0.0f : q.s * exp2f(base(q.m) - c))};
    };
#pragma unroll
    for (int d = 32; d >= kJoinTokens; d >>= 1) p = merge(p, Lse{__shfl_xor(p.m, d), __shfl_xor(p.s, d)});
    if ((threadIdx.x & 63) < kJoinTokens) waves[threadIdx.x >> 6][t] = p;
    __syncthreads();
    if (threadIdx.x >= kJoinTokens || token >= tokens) return;
#pragma unroll
    for (int w = 1; w < kJoinThreads / 64; ++w) p = merge(p, waves[w][t]);
    if (kind != kValid) {
        lse2[token] = logp[token] = kind == kIgnored ? 0.0f : __builtin_nanf("");
        return;
    }
    const float c = base(p.m), l = log2f(p.s);
    lse2[token] = c + l;
    logp[token] = (fmaf(target[token], scale2, -c) - l) * kLn2;
}

// ---------------------------------------------------------------------
// fp32 logits that a library product has left: kT lanes per row, one pass, each
// lane with its own running maximum and sum.  Bound by the read, 4.9 to 6.5 TB/s
// (part of it from cache) from 1,000 words on.  us at 16 | 64 | 256 | 1024 lanes,
// 1 GiB of logits: 512 words 180 | 308 | 967 | 2924, 1024 189 | 174 | 686 | 1498,
// 4096 193 | 180 | 188 | 617, 8192 206 | 187 | 167 | 317, 16384 192 | 196 | 178 |
// 174, 32000 236 | 201 | 183 | 164; 64 rows of 16384 45 | 14 | 5.8 | 5.2.
// ---------------------------------------------------------------------
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

// ---------------------------------------------------------------------
// Gradients.  What multiplies each row: grad * scale * (1 - p_y), and, of fp16
// operands, a power of two that brings the largest of them into [1/2, 1): a mean
// over many tokens leaves them near fp16's least numbers, and a hidden row times
// a factor below 1 is finite in fp16 whenever the row is.  One workgroup.
// ---------------------------------------------------------------------
struct Weights {
    const float *grad, *logp;
    const int64_t* labels;
    int64_t ignore_index;
    uint64_t n;
    uint32_t vocab;
    float scale;
    float* weight;
    float* norm;   // or null
    float unlift;  // what takes D's kLift out
    bool normalise;
    __device__ float operator()(uint64_t i) const {
        const float g = grad[i];
        const RowKind kind = row_kind(labels[i], ignore_index, vocab);
        if (kind == kIgnored || g == 0.0f) return 0.0f;
        return kind == kValid ? g * scale * rest_of(logp[i]) : __builtin_nanf("");
    }
};

constexpr int kWeightThreads = 1024;
__global__ __launch_bounds__(kWeightThreads) void logps_weight_kernel(const Weights a) {
    row_weights<kWeightThreads>(a, blockIdx.x, gridDim.x);
}

// D from what the product kept, in place.  A workgroup takes 4,096 words of a
// token, 16 bytes at a time.  A token without a gradient of its own, masked ones
// above all, has D = 0 whatever its hidden states hold, and is not read; rows
// from `tokens` on are cleared (they pad the weight gradient's sum).  The launch's
// first `others` workgroups make the rows' weights, which nothing here needs.
// Bound by its bytes, 2.1 GB at 4092 tokens of 128256 words: 0.32 ms with all of
// them, 6.6 TB/s, part of it from the last-level cache.
constexpr int kGradThreads = 256;
constexpr int kKeepColumns = kGradThreads * kGroup * 2;
template <typename Fmt>
__global__ __launch_bounds__(kGradThreads) void logps_keep_grad_kernel(uint16_t* __restrict__ keep, uint64_t ld,
                                                                       uint32_t tokens, uint32_t vocab,
                                                                       uint32_t col_blocks, uint64_t first,
                                                                       const float2* __restrict__ parts,
                                                                       const int64_t* __restrict__ labels,
                                                                       int64_t ignore_index,
                                                                       const float* __restrict__ lse2,
                                                                       const float* __restrict__ logp,
                                                                       const float* __restrict__ grad,
                                                                       const Weights weights, uint32_t others) {
    if (blockIdx.x < others) return row_weights<kGradThreads>(weights, blockIdx.x, others);
    const uint64_t b = first + blockIdx.x - others, row = b / col_blocks;
    const uint32_t col = uint32_t(b % col_blocks) * kKeepColumns + threadIdx.x * kGroup;
    uint16_t* k = keep + row * ld;
    const int64_t y = row < tokens ? labels[row] : ignore_index;
    const RowKind kind = row < tokens && grad[row] == 0.0f ? kIgnored : row_kind(y, ignore_index, vocab);
    if (row >= tokens || kind != kValid) {
        const uint32_t w = row < tokens && kind == kBadLabel ? Fmt::kNan2 : 0u;
#pragma unroll
        for (int j = 0; j < 2; ++j)
            if (col + j * kGradThreads * kGroup < ld)
                *reinterpret_cast<u32x4*>(k + col + j * kGradThreads * kGroup) = u32x4{w, w, w, w};
        return;
    }
    const float l = lse2[row], by = -1.0f / rest_of(logp[row]);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const uint32_t c = col + j * kGradThreads * kGroup;
        if (c >= ld) break;
        u32x4* p = reinterpret_cast<u32x4*>(k + c);
        const u32x4 v = *p;
        const float f = exp2f(base(parts[uint64_t(c / kSpan) * tokens + row].x) - l) * by;
        u32x4 o;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = Fmt::pack(lifted<Fmt>(Fmt::lo(v[i]) * f), lifted<Fmt>(Fmt::hi(v[i]) * f));
        *p = o;
        // over what this lane has just stored
        if (uint64_t(y) - c < uint64_t(kGroup)) k[y] = uint16_t(Fmt::pack(kLift<Fmt>, 0.0f));
    }
}

// The hidden gradient of a few tokens, row weight * (D W), in one launch.  A
// workgroup takes 16 tokens and 128 of the hidden dimensions, its waves the words
// in turns of 32.  The words are the sum's dimension here and W's rows lie along
// the other: a lane reads 8 neighbouring dimensions of 8 words and turns them
// around in registers, so that its operand for dimension j of the 8 is one
// register from each pair of words, and it ends up with 8 neighbours of a token.
// No LDS but for the waves' sums.  Inside a backward 17.5 us at 126 x 512 x 4096,
// 18.4 at 128 x 2048 x 4096, 33.4 at 250 x 4096 x 4096: the waits for W's words bind
// it, about 1 us a turn of 256, whatever is on its way (launched again and again on
// operands that stay in the caches 14, 15 and 32, where 16 waves or 64 dimensions a
// workgroup took 14 and 13 at the first).  A call this small waits longer for the
// host.
constexpr int kHgWaves = 8;
constexpr int kHgTokens = 16;
constexpr int kHgColumns = 128;
template <typename Fmt>
__global__ __launch_bounds__(kHgWaves * 64, 2) void logps_hidden_grad_kernel(
    const uint16_t* __restrict__ d, uint64_t ld, uint32_t tokens, const uint16_t* __restrict__ weight, uint64_t ldw,
    uint32_t vocab, uint32_t cols, uint32_t col_blocks, const float* __restrict__ by, const float* __restrict__ norm,
    uint16_t* __restrict__ out) {
    constexpr uint32_t kWords = 32;
    __shared__ float sums[kHgWaves][32][64];
    const uint32_t lane = threadIdx.x & 63, l16 = lane & 15, quad = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t token0 = blockIdx.x / col_blocks * kHgTokens;
    const uint32_t col = blockIdx.x % col_blocks * kHgColumns + l16 * 8;
    const uint32_t from = col < cols ? col : 0;   // columns past the last are not stored
    const uint16_t* dp = d + uint64_t(token0 + l16) * ld;

    struct Words {
        u32x4 d, w[8];
    };
    const auto load = [&](uint32_t v) {
        Words x;
        v += quad * 8;
        x.d = *reinterpret_cast<const u32x4*>(dp + v);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            x.w[i] = v + i < vocab ? *reinterpret_cast<const u32x4*>(weight + (v + i) * ldw + from) : u32x4{0, 0, 0, 0};
        return x;
    };
    f32x4 acc[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const auto add = [&](const Words& x) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            u32x4 b;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                b[i] = __builtin_amdgcn_perm(x.w[2 * i + 1][j / 2], x.w[2 * i][j / 2], j % 2 ? 0x07060302u : 0x05040100u);
            acc[j] = mfma(Fmt{}, x.d, b, acc[j]);
        }
    };
    // the next words are on their way while these are used (four turns on their way
    // took twice the registers and gave 5 % at 16384 words, none at 4096)
    constexpr uint32_t kTurn = kHgWaves * kWords;
    uint32_t v = wave * kWords;
    if (v < vocab) {
        Words x = load(v);
        for (; v + kTurn < vocab; v += kTurn) {
            const Words next = load(v + kTurn);
            add(x);
            x = next;
        }
        add(x);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[wave][j * 4 + i][lane] = acc[j][i];
    __syncthreads();
    // a wave takes one of a lane's four tokens and half of its columns
    static_assert(kHgWaves == 8, "four tokens, two halves");
    const uint32_t i = wave / 2, j0 = wave % 2 * 4, token = token0 + quad * 4 + i;
    f32x4 t;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float s[kHgWaves];
#pragma unroll
        for (int w = 0; w < kHgWaves; ++w) s[w] = sums[w][(j0 + j) * 4 + i][lane];
        t[j] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
    }
    if (token >= tokens || col >= cols) return;
    const float f = by[token];
    t = f == 0.0f ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : t * f * (norm != nullptr ? *norm : 1.0f);
    uint32_t* o = reinterpret_cast<uint32_t*>(out + uint64_t(token) * cols + col + j0);
    o[0] = Fmt::pack(t[0], t[1]), o[1] = Fmt::pack(t[2], t[3]);
}

// The weight gradient of up to 256 tokens, D^T times the weighted hidden rows: an
// outer product with a short sum, which its output's bytes bound: 64 x 4096 x
// 128256, 1.05 GB, 219 us, 4.8 TB/s (a fill of that size reaches 6.9), a library's
// product 362; 256 x 4096 x 128256 288 | 464, 128 x 768 x 50257 20 | 31, 200 x 1024
// x 32000 30 | 32.  A workgroup takes 256 words, each wave 64 with all their
// tokens as operands in registers, and goes along the hidden dimensions 128 at a
// time; the hidden rows of those, transposed, come through LDS in the order in
// which lanes read them, the next ones while these are used.  The words of D lie
// side by side, so a lane reads 4 of them of 8 tokens and turns them around; word
// l and dimension l of an operand are 4 l + i and 8 l + j of the wave's 64 and
// 128, so that a lane ends up with 8 neighbours of a word, 16 lanes with 256
// bytes.  Over 128 tokens the operands take half of a wave's registers and the
// dimensions go 64 at a time, which leaves room for a second workgroup: 256 x
// 4096 x 128256 288 us, alone and 128 at a time 357.
constexpr int kWgThreads = 256;
constexpr size_t kWgTokens = 256;
constexpr int kWgWords = 256;
template <int kSteps>   // tokens / 32, padded
constexpr int kWgLane = kSteps > 4 ? 4 : 8;   // neighbouring dimensions of a lane
template <typename Fmt, int kSteps>
__global__ __launch_bounds__(kWgThreads, 2) void logps_weight_grad_kernel(
    const uint16_t* __restrict__ d, uint64_t ld, uint32_t vocab, const uint16_t* __restrict__ hidden_t, uint32_t cols,
    uint32_t runs, uint32_t per, const float* __restrict__ norm, uint16_t* __restrict__ out) {
    constexpr uint32_t kTokens = kSteps * 32;
    constexpr int kWaves = kWgThreads / 64, kFW = 4, kFH = kWgLane<kSteps>, kColumns = 16 * kFH;
    using Piece = std::conditional_t<kFH == 8, u32x4, u32x2>;
    constexpr int kPieces = kFH * kSteps;   // of 1 KB: an operand of a wave
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2][kPieces * 1024];
    const uint32_t lane = threadIdx.x & 63, l16 = lane & 15, quad = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t word0 = blockIdx.x / runs * kWgWords + wave * 64;
    const uint32_t first = blockIdx.x % runs * per, last = min(first + per, (cols + kColumns - 1) / kColumns);

    typedef __attribute__((address_space(3))) uint8_t Lds;
    typedef const __attribute__((address_space(1))) uint8_t Global;
    // Rows past the last are the last one again and are not stored.
    const auto copy = [&](uint32_t block, uint32_t buf) {
#pragma unroll
        for (int k = 0; k < kPieces / kWaves; ++k) {
            const uint32_t piece = k * kWaves + wave, j = piece / kSteps, s = piece % kSteps;
            const uint32_t row = min(block * kColumns + l16 * kFH + j, cols - 1);
            __builtin_amdgcn_global_load_lds((Global*)(hidden_t + uint64_t(row) * kTokens + s * 32 + quad * 8),
                                             (Lds*)(&lds[buf][piece * 1024]), 16, 0, 0);
        }
    };
    const auto meet = [] {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0x0070);
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    copy(first, 0);
    u32x4 a[kFW][kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
        u32x2 x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            x[i] = *reinterpret_cast<const u32x2*>(d + (s * 32 + quad * 8 + i) * ld +
                                                   min(word0 + l16 * 4, uint32_t(ld) - 4));
#pragma unroll
        for (int w = 0; w < kFW; ++w)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                a[w][s][i] = __builtin_amdgcn_perm(x[2 * i + 1][w / 2], x[2 * i][w / 2], w % 2 ? 0x07060302u : 0x05040100u);
    }
    const float scale = norm != nullptr ? *norm : 1.0f;
    meet();
    for (uint32_t block = first; block < last; ++block) {
        const uint32_t buf = (block - first) & 1;
        if (block + 1 < last) copy(block + 1, buf ^ 1);
        f32x4 acc[kFW][kFH];
#pragma unroll
        for (int w = 0; w < kFW; ++w)
#pragma unroll
            for (int j = 0; j < kFH; ++j) acc[w][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < kFH; ++j)
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                const u32x4 b = *reinterpret_cast<const u32x4*>(&lds[buf][(j * kSteps + s) * 1024 + lane * 16]);
#pragma unroll
                for (int w = 0; w < kFW; ++w) acc[w][j] = mfma(Fmt{}, a[w][s], b, acc[w][j]);
            }
        // the next rows are there, and these are not read again
        meet();
        const uint32_t col = block * kColumns + l16 * kFH;
        if (col >= cols) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int w = 0; w < kFW; ++w) {
                const uint32_t word = word0 + (quad * 4 + i) * 4 + w;
                Piece o;
#pragma unroll
                for (int j = 0; j < kFH / 2; ++j) o[j] = Fmt::pack(acc[w][2 * j][i] * scale, acc[w][2 * j + 1][i] * scale);
                if (word < vocab) *reinterpret_cast<Piece*>(out + uint64_t(word) * cols + col) = o;
            }
    }
}

// The gradients' large products, 256 x 256 outputs a workgroup.  Both have one
// operand whose rows lie along the sum (X: D's tokens for the hidden gradient, the
// transposed hidden rows for the weight gradient) and one whose rows lie across it
// (Y: W, D).  X goes through LDS as the forward's operands do; Y's rows of 256
// columns go there as they lie and are read four rows at once, transposed, by
// ds_read_b64_tr_b16.  Its 32-byte granules are swizzled by the row, so that the 16
// rows of a wave's read take every bank twice, the least there is.  The copies,
// reads and products go on as in the forward's kernel; LDS, 96 KB read and 32 KB
// written for every 32 terms, is as busy as the matrix cores.  us, a library's
// product | this: hidden gradient 8190 x 5120 x 152064 in two parts 9655 | 9473,
// 4092 x 4096 x 128256 3049 | 3034, 2046 x 2560 x 151936 1806 | 1310, 4000 x 3584 x
// 152064 3319 | 3484; weight gradient, bf16 and fp16 (there into fp32, still to be
// scaled), 500 x 4096 x 128256 714, 1045 | 679, 8190 x 2560 x 50257 1732, 2101 |
// 1597, 4092 x 4096 x 128256 3219 bf16 | 3310.  Four waves of 128 x 128 outputs
// read a third less from LDS, but one wave a SIMD leaves its waits open: 3900.
struct Product {
    const uint16_t* x;   // [rows, 64 steps], ldx
    const uint16_t* y;   // [sum, cols], ldy, of which wide may be read
    uint32_t ldx, ldy, rows, cols, wide, sum;
    uint32_t steps, each;   // 64 terms each: in all and in a part
    void* out;
    const float* norm;
    uint32_t parts;         // with live, of the hidden gradient: at most
    const int32_t* live;    // or null: how many tokens there are, of rows or of sum
};
constexpr int kPrTile = 256;
typedef short Four __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) Four LdsFour;
// restrict: or the compiler waits for every copy into LDS before this read
__device__ __forceinline__ u32x2 read_turned(LdsFour* __restrict__ p) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(p));
}
template <typename Fmt, bool kHidden>   // out: fp32 [parts, rows, cols], or 16-bit [cols, rows]
__global__ __launch_bounds__(512, 2) void logps_product_kernel(const Product a) {
    constexpr int kWP = 2, kWQ = 4, kFP = 8, kFQ = 4, kWaves = kWP * kWQ;
    constexpr int kBuffer = 2 * kPrTile * kRowBytes, kLX = kPrTile / 8 / kWaves, kLY = kTerms / 2 / kWaves;
    constexpr int kTurnRow = kFP * 32;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * kBuffer];
    const uint32_t lane = threadIdx.x & 63, l16 = lane & 15, quad = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t wp = wave / kWQ, wq = wave % kWQ;

    // As in the forward: each XCD has a contiguous run, 8 tiles of rows beside each other; tiles
    // and terms without a token are left out.
    const uint32_t live = a.live != nullptr ? uint32_t(*a.live) : ~0u;
    const uint32_t rows = kHidden ? min(a.rows, live) : a.rows;
    const uint32_t all = kHidden || a.live == nullptr ? a.steps : min(a.steps, max((live + kTerms - 1) / kTerms, 1u));
    const uint32_t tiles_p = (rows + kPrTile - 1) / kPrTile, tiles_q = (a.cols + kPrTile - 1) / kPrTile;
    uint32_t parts = a.parts, each = a.each;
    if (kHidden && a.live != nullptr) parts = parts_of_rows(rows, a.cols, a.steps, a.parts), each = (a.steps + parts - 1) / parts;
    const uint32_t tiles = tiles_p * tiles_q * parts, xcd = blockIdx.x % 8, run = tiles / 8, more = tiles % 8;
    if (blockIdx.x / 8 >= run + (xcd < more)) return;
    uint32_t id = xcd * run + min(xcd, more) + blockIdx.x / 8;
    const uint32_t part = id / (tiles_p * tiles_q);
    id -= part * tiles_p * tiles_q;
    const uint32_t first_p = id / (kGroupT * tiles_q) * kGroupT, group = min(uint32_t(kGroupT), tiles_p - first_p);
    const uint32_t in = id - first_p * tiles_q;
    const uint32_t q0 = in / group * kPrTile, p0 = (first_p + in % group) * kPrTile;
    const uint32_t step0 = part * each, steps = min(all - step0, each);

    const uint8_t* gx = reinterpret_cast<const uint8_t*>(a.x + uint64_t(p0) * a.ldx + uint64_t(step0) * kTerms);
    const uint8_t* gy = reinterpret_cast<const uint8_t*>(a.y + uint64_t(step0) * kTerms * a.ldy + q0);
    const uint64_t y_step = uint64_t(a.ldy) * (2 * kTerms);
    uint32_t off_x[kLX], row_y[kLY], col_y[kLY];
#pragma unroll
    for (int j = 0; j < kLX; ++j)
        off_x[j] = min((j * kWaves + wave) * 8 + (lane >> 3), rows - 1 - p0) * (a.ldx * 2) +
                   ((lane & 7) ^ (lane >> 3)) * 16;
#pragma unroll
    for (int j = 0; j < kLY; ++j) {
        const uint32_t row = (j * kWaves + wave) * 2 + (lane >> 5), chunk = lane & 31;
        const uint32_t from = ((chunk >> 1 ^ (row & 3) ^ (row >> 3 & 1) << 2) << 1 | (chunk & 1)) * 8;
        row_y[j] = row;
        col_y[j] = min(from, a.wide - 8 - q0) * 2;   // columns past the last are not stored
    }
    typedef __attribute__((address_space(3))) uint8_t Lds;
    typedef const __attribute__((address_space(1))) uint8_t Global;
    const auto copy = [&](uint32_t step, uint32_t buf) {
        uint8_t* to = lds + buf * kBuffer + wave * 1024;
#pragma unroll
        for (int j = 0; j < kLX; ++j)
            __builtin_amdgcn_global_load_lds((Global*)(gx + step * kRowBytes + off_x[j]), (Lds*)(to + j * kWaves * 1024),
                                             16, 0, 0);
        // rows past the sum's end are its last: X has zeros there
        const uint32_t last = a.sum - 1 - (step0 + step) * kTerms;
#pragma unroll
        for (int j = 0; j < kLY; ++j)
            __builtin_amdgcn_global_load_lds((Global*)(gy + step * y_step + min(row_y[j], last) * (a.ldy * 2) + col_y[j]),
                                             (Lds*)(to + kPrTile * kRowBytes + j * kWaves * 1024), 16, 0, 0);
    };
    const uint32_t at = (quad ^ (l16 & 7)) * 16, at_x = (wp * kFP * 16 + l16) * kRowBytes;
    const uint32_t turn_y = (l16 >> 2) | (quad & 1) << 2;
    const uint32_t at_y = kPrTile * kRowBytes + (quad * 8 + (l16 >> 2)) * (kPrTile * 2) + (l16 & 3) * 8;
    u32x4 x[2][kFP], y[2][kFQ];
    const auto read = [&](uint32_t buf, int half) {
        const uint8_t* from = lds + buf * kBuffer;
#pragma unroll
        for (int i = 0; i < kFP; ++i)
            x[half][i] = *reinterpret_cast<const u32x4*>(from + (at ^ (half * 64)) + at_x + i * 16 * kRowBytes);
#pragma unroll
        for (int j = 0; j < kFQ; ++j) {
            const uint8_t* p = from + at_y + half * 32 * (kPrTile * 2) + (((wq * kFQ + j) ^ turn_y) * 32);
            const u32x2 lo = read_turned((LdsFour*)p), hi = read_turned((LdsFour*)(p + 4 * kPrTile * 2));
            y[half][j] = u32x4{lo.x, lo.y, hi.x, hi.y};
        }
    };
    f32x4 acc[kFP][kFQ];
    const auto multiply = [&](int half) {
#pragma unroll
        for (int i = 0; i < kFP; ++i)
#pragma unroll
            for (int j = 0; j < kFQ; ++j)
                acc[i][j] = kHidden ? mfma(Fmt{}, y[half][j], x[half][i], acc[i][j])
                                    : mfma(Fmt{}, x[half][i], y[half][j], acc[i][j]);
    };
    const auto meet = [] {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0x0070);
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    const auto step = [&](uint32_t s, auto kMore) {
        read(s & 1, 1);
        multiply(0);
        interleave<kFP + 2 * kFQ, kFP * kFQ, 0>();
        meet();
        if constexpr (decltype(kMore)::value) copy(s + 2, s & 1);
        read((s + 1) & 1, 0);
        multiply(1);
        interleave<kFP + 2 * kFQ, kFP * kFQ, decltype(kMore)::value ? kLX + kLY : 0>();
        __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (int i = 0; i < kFP; ++i)
#pragma unroll
        for (int j = 0; j < kFQ; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    copy(0, 0);
    if (steps > 1) copy(1, 1);
    meet();
    read(0, 0);
    uint32_t s = 0;
    for (; s + 2 < steps; ++s) step(s, std::true_type{});
    if (s + 1 < steps) step(s++, std::false_type{});
    read(s & 1, 1);
    multiply(0);
    meet();   // the buffers are not read again
    multiply(1);
    if constexpr (kHidden) {
        float* out = static_cast<float*>(a.out) + uint64_t(part) * a.rows * a.cols;
#pragma unroll
        for (int i = 0; i < kFP; ++i) {
            const uint32_t row = p0 + wp * kFP * 16 + i * 16 + l16;
            if (row >= rows) continue;
#pragma unroll
            for (int j = 0; j < kFQ; ++j) {
                const uint32_t col = q0 + wq * kFQ * 16 + j * 16 + quad * 4;
                if (col < a.cols) *reinterpret_cast<f32x4*>(out + uint64_t(row) * a.cols + col) = acc[i][j];
            }
        }
    } else {
        const float scale = a.norm != nullptr ? *a.norm : 1.0f;
        uint16_t* out = static_cast<uint16_t*>(a.out);
        uint8_t* const turn = lds + wave * 16 * kTurnRow;
#pragma unroll
        for (int j = 0; j < kFQ; ++j) {
#pragma unroll
            for (int i = 0; i < kFP; ++i) {
                const f32x4 e = acc[i][j] * scale;
                const uint32_t to = ((i * 2 + (quad >> 1)) ^ l16) * 16 + (quad & 1) * 8;
                *reinterpret_cast<u32x2*>(turn + l16 * kTurnRow + to) = u32x2{Fmt::pack(e[0], e[1]), Fmt::pack(e[2], e[3])};
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t at_row = k * 4 + quad;
                const u32x4 o = *reinterpret_cast<const u32x4*>(turn + at_row * kTurnRow + (l16 ^ at_row) * 16);
                const uint32_t col = q0 + wq * kFQ * 16 + j * 16 + at_row, row = p0 + wp * kFP * 16 + l16 * 8;
                if (col < a.cols && row < a.rows) *reinterpret_cast<u32x4*>(out + uint64_t(col) * a.rows + row) = o;
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
    }
}

// Rows times their weights, 0 where that is whatever the row holds.  Bound by its
// bytes; as separate operations it is three launches.
template <typename Fmt>
__global__ __launch_bounds__(kGradThreads) void logps_weighted_kernel(const uint16_t* __restrict__ hidden, uint64_t ldh,
                                                                      uint32_t groups, uint32_t cols, uint64_t first,
                                                                      uint64_t count, const float* __restrict__ by,
                                                                      uint16_t* __restrict__ out) {
    const uint64_t i = (first + blockIdx.x) * kGradThreads + threadIdx.x;
    if (i >= count) return;
    const uint64_t row = i / groups;
    const uint32_t col = uint32_t(i - row * groups) * kGroup;
    const float f = by[row];
    u32x4 o = {0, 0, 0, 0};
    if (f != 0.0f) {
        const u32x4 v = *reinterpret_cast<const u32x4*>(hidden + row * ldh + col);
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = Fmt::pack(Fmt::lo(v[j]) * f, Fmt::hi(v[j]) * f);
    }
    *reinterpret_cast<u32x4*>(out + row * cols + col) = o;
}

// D from fp32 logits; a workgroup takes 1,024 words of a row.
constexpr int kGradColumns = 1024;
struct Out32 {
    using S = float;
    static constexpr float kTop = 1.0f;
    __device__ static void store(S* p, float f) { *p = f; }
};
template <typename Fmt>
struct Out16 {
    using S = uint16_t;
    static constexpr float kTop = kLift<Fmt>;
    __device__ static void store(S* p, float f) { *p = uint16_t(Fmt::pack(lifted<Fmt>(f), 0.0f)); }
};
template <typename Out>
__global__ __launch_bounds__(kGradThreads) void logps_grad_kernel(const float* logits, uint64_t ld, uint32_t vocab,
                                                                  uint32_t col_blocks, uint64_t first,
                                                                  const int64_t* __restrict__ labels,
                                                                  int64_t ignore_index, float scale,
                                                                  const float* __restrict__ lse,
                                                                  const float* __restrict__ logp,
                                                                  const float* __restrict__ grad,
                                                                  typename Out::S* dz, uint64_t ld_dz) {
    const uint64_t b = first + blockIdx.x, row = b / col_blocks;
    const uint32_t col = uint32_t(b % col_blocks) * kGradColumns + threadIdx.x;
    const int64_t y = labels[row];
    const RowKind kind = grad[row] == 0.0f ? kIgnored : row_kind(y, ignore_index, vocab);
    const float* x = logits + row * ld;
    typename Out::S* o = dz + row * ld_dz;
    const float l = lse[row], by = -Out::kTop / rest_of(logp[row]);
#pragma unroll
    for (int k = 0; k < kGradColumns / kGradThreads; ++k) {
        const uint32_t j = col + k * kGradThreads;
        if (j >= vocab) break;
        float f = kind == kIgnored ? 0.0f : __builtin_nanf("");
        if (kind == kValid) f = int64_t(j) == y ? Out::kTop : expf(x[j] * scale - l) * by;
        Out::store(o + j, f);
    }
}

// ---------------------------------------------------------------------
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

template <typename Fmt, int kSteps>
int launch_weight_grad(const void* d, size_t ld, size_t vocab, const void* hidden_t, size_t cols, const float* norm,
                       void* out, hipStream_t st) {
    // Runs along the hidden dimensions: what fits one round of two workgroups a
    // compute unit, and with too many words for that 1,024 workgroups.  us at one
    // round | two, 256 x 768 x 50257 30 | 40, 200 x 2048 x 50257 59 | 72; at about
    // 500 | 1,000 | 1,500 workgroups, 64 x 4096 x 128256 239 | 262 | 219, 256 x 4096 x
    // 128256 316 | 331 | 288.
    constexpr uint32_t kColumns = 16 * kWgLane<kSteps>;
    const uint32_t groups = uint32_t((vocab + kWgWords - 1) / kWgWords);
    const uint32_t blocks = uint32_t((cols + kColumns - 1) / kColumns);
    const uint32_t want = groups <= 256 ? 512 / groups : (1024 + groups - 1) / groups;
    const uint32_t per = (blocks + want - 1) / want, runs = (blocks + per - 1) / per;
    hipLaunchKernelGGL((logps_weight_grad_kernel<Fmt, kSteps>), dim3(groups * runs), dim3(kWgThreads), 0, st,
                       static_cast<const uint16_t*>(d), uint64_t(ld), uint32_t(vocab),
                       static_cast<const uint16_t*>(hidden_t), uint32_t(cols), runs, per, norm,
                       static_cast<uint16_t*>(out));
    return status();
}

template <typename Fmt>
int dispatch_weight_grad(const void* d, size_t ld, size_t tokens, size_t vocab, const void* hidden_t, size_t cols,
                         const float* norm, void* out, hipStream_t st) {
    switch (tokens / 64) {
        case 1: return launch_weight_grad<Fmt, 2>(d, ld, vocab, hidden_t, cols, norm, out, st);
        case 2: return launch_weight_grad<Fmt, 4>(d, ld, vocab, hidden_t, cols, norm, out, st);
        case 3: return launch_weight_grad<Fmt, 6>(d, ld, vocab, hidden_t, cols, norm, out, st);
        default: return launch_weight_grad<Fmt, 8>(d, ld, vocab, hidden_t, cols, norm, out, st);
    }
}

template <bool kHidden>
int launch_product(const Product& a, uint32_t parts, int dtype, hipStream_t st) {
    const uint64_t tiles = uint64_t((a.rows + kPrTile - 1) / kPrTile) * ((a.cols + kPrTile - 1) / kPrTile) * parts;
    if (tiles > kMaxLanes / 512) return SF_EINVAL;
    const auto kernel = dtype == SF_DTYPE_BF16 ? logps_product_kernel<Bf16, kHidden> : logps_product_kernel<F16, kHidden>;
    hipLaunchKernelGGL(kernel, dim3(uint32_t(tiles)), dim3(512), 0, st, a);
    return status();
}

// kernel(first, blocks) in as many launches as `blocks` workgroups need.
template <typename Launch>
int in_launches(uint64_t blocks, Launch launch) {
    constexpr uint64_t kMax = kMaxLanes / kGradThreads;
    for (uint64_t first = 0; first < blocks; first += kMax) {
        launch(first, uint32_t(blocks - first < kMax ? blocks - first : kMax));
        const int e = status();
        if (e != SF_OK) return e;
    }
    return SF_OK;
}

template <typename Out>
int launch_grad(const float* x, uint64_t ld, uint64_t rows, uint32_t vocab, const int64_t* labels, int64_t ignore,
                float scale, const float* lse, const float* logp, const float* grad, void* dz, uint64_t ld_dz,
                hipStream_t st) {
    const uint32_t col_blocks = (vocab + kGradColumns - 1) / kGradColumns;
    return in_launches(rows * col_blocks, [&](uint64_t first, uint32_t blocks) {
        hipLaunchKernelGGL(logps_grad_kernel<Out>, dim3(blocks), dim3(kGradThreads), 0, st, x, ld, vocab, col_blocks,
                           first, labels, ignore, scale, lse, logp, grad, static_cast<typename Out::S*>(dz), ld_dz);
    });
}

bool sizes_bad(size_t rows, size_t vocab) {
    return vocab == 0 || vocab > (size_t(1) << 30) || rows >= (size_t(1) << 31);
}

int hidden_product(const void* d, size_t ld, size_t rows, const int32_t* live, const void* weight, size_t ldw, size_t vocab,
                   size_t cols, int nparts, float* parts, int dtype, sf_stream_t stream) {
    if (rows == 0) return SF_OK;
    if (d == nullptr || weight == nullptr || parts == nullptr || sizes_bad(rows, vocab) || cols == 0 ||
        cols > (size_t(1) << 22) || ld < (vocab + kTerms - 1) / kTerms * kTerms || ld > (size_t(1) << 22) || ldw < cols ||
        ldw > (size_t(1) << 22) || nparts < 1 || size_t(nparts) > (vocab + kTerms - 1) / kTerms)
        return SF_EINVAL;
    if (dtype != SF_DTYPE_BF16 && dtype != SF_DTYPE_F16) return SF_EDTYPE;
    if (cols % 8 != 0 || ld % 8 != 0 || ldw % 8 != 0 || misaligned(d, 16) || misaligned(weight, 16) || misaligned(parts, 16))
        return SF_EALIGN;
    Product a = {static_cast<const uint16_t*>(d), static_cast<const uint16_t*>(weight), uint32_t(ld), uint32_t(ldw),
                 uint32_t(rows), uint32_t(cols), uint32_t(cols), uint32_t(vocab),
                 uint32_t((vocab + kTerms - 1) / kTerms), 0, parts, nullptr, uint32_t(nparts), live};
    a.each = (a.steps + nparts - 1) / nparts;
    if ((a.steps + a.each - 1) / a.each != uint32_t(nparts)) return SF_EINVAL;
    return launch_product<true>(a, nparts, dtype, reinterpret_cast<hipStream_t>(stream));
}

int weight_grad(const void* d, size_t ld, size_t tokens, const int32_t* live, size_t vocab, const void* hidden_t, size_t cols,
                const float* norm, int dtype, void* out, sf_stream_t stream) {
    if (d == nullptr || hidden_t == nullptr || out == nullptr || sizes_bad(tokens, vocab) || tokens == 0 ||
        tokens > (size_t(1) << 22) || cols == 0 || cols > (size_t(1) << 22) || ld < vocab || ld > (size_t(1) << 22))
        return SF_EINVAL;
    if (dtype != SF_DTYPE_BF16 && dtype != SF_DTYPE_F16) return SF_EDTYPE;
    if (tokens % 64 != 0 || cols % 8 != 0 || ld % 8 != 0 || misaligned(d, 16) || misaligned(hidden_t, 16) ||
        misaligned(out, 16))
        return SF_EALIGN;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (tokens > kWgTokens || live != nullptr) {
        const uint32_t steps = uint32_t(tokens / kTerms);
        const Product a = {static_cast<const uint16_t*>(hidden_t), static_cast<const uint16_t*>(d), uint32_t(tokens),
                           uint32_t(ld), uint32_t(cols), uint32_t(vocab), uint32_t(ld), uint32_t(tokens), steps, steps,
                           out, norm, 1, live};
        return launch_product<false>(a, 1, dtype, st);
    }
    return dtype == SF_DTYPE_BF16 ? dispatch_weight_grad<Bf16>(d, ld, tokens, vocab, hidden_t, cols, norm, out, st)
                                  : dispatch_weight_grad<F16>(d, ld, tokens, vocab, hidden_t, cols, norm, out, st);
}

}  // namespace

extern "C" {

int sf_logps_tiles(const void* weight, size_t ldw, size_t vocab, const void* hidden, size_t ldh, size_t rows,
                   size_t hidden_size, const int64_t* labels, int64_t ignore_index, float scale, int dtype, void* parts,
                   float* target, int32_t* order, void* keep, size_t ld_keep, float* lse2, float* logp,
                   sf_stream_t stream) {
    if (rows == 0) return SF_OK;
    if (weight == nullptr || hidden == nullptr || labels == nullptr || parts == nullptr || target == nullptr ||
        lse2 == nullptr || logp == nullptr || sizes_bad(rows, vocab))
        return SF_EINVAL;
    // 32-bit byte offsets inside a tile of 256 rows
    constexpr size_t kMostLd = size_t(1) << 22;
    if (hidden_size == 0 || ldw < hidden_size || ldh < hidden_size || ldw > kMostLd || ldh > kMostLd || !(scale > 0.0f))
        return SF_EINVAL;
    if (dtype != SF_DTYPE_BF16 && dtype != SF_DTYPE_F16) return SF_EDTYPE;
    const size_t spans = (vocab + kSpan - 1) / kSpan;
    if (keep != nullptr && ld_keep < spans * kSpan) return SF_EINVAL;
    if (hidden_size % kTerms != 0 || ldw % kGroup != 0 || ldh % kGroup != 0 || misaligned(weight, 16) ||
        misaligned(hidden, 16) || misaligned(parts, 8) || misaligned(keep, 16) || ld_keep % kGroup != 0)
        return SF_EALIGN;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (order != nullptr && uint64_t(rows) * ldh * 2 > UINT32_MAX) return SF_ETOOBIG;   // 32-bit byte offsets of all rows
    // Rows of one launch: whole tiles of 256, as many as its lanes allow for the
    // product (2.1 M rows of 128256 words) and the join.
    constexpr uint64_t kTile = 256, kMostRows = kMaxLanes / kJoinThreads * kJoinTokens;
    const uint64_t fit = kMaxLanes / kTileKinds[0].lanes / spans * kTile, most = fit < kMostRows ? fit : kMostRows;
    for (uint64_t r = 0; r < rows; r += most) {
        const uint32_t n = uint32_t(rows - r < most ? rows - r : most);
        const Tiles a = {static_cast<const uint16_t*>(weight), static_cast<const uint16_t*>(hidden) + r * ldh,
                         uint32_t(ldw), uint32_t(ldh), uint32_t(vocab), n, uint32_t(hidden_size / kTerms), labels + r,
                         order == nullptr ? nullptr : order + r, scale * kLog2e, static_cast<float2*>(parts) + r, rows,
                         target + r, keep == nullptr ? nullptr : static_cast<uint16_t*>(keep) + r * ld_keep, ld_keep,
                         nullptr, nullptr, nullptr, 0, false};
        int e = SF_OK;
        if (order != nullptr) {   // its last element is the next launch's first, which is written behind this one's
            hipLaunchKernelGGL(logps_order_kernel<HasLabel>, dim3(1), dim3(kOrderThreads), 0, st,
                               HasLabel{a.labels, ignore_index, a.vocab}, n, order + r);
            e = status();
            if (e != SF_OK) return e;
        }
        e = dtype == SF_DTYPE_BF16 ? dispatch_tiles<Bf16, false>(a, st) : dispatch_tiles<F16, false>(a, st);
        if (e != SF_OK) return e;
        hipLaunchKernelGGL(logps_join_kernel, dim3((n + kJoinTokens - 1) / kJoinTokens), dim3(kJoinThreads), 0, st,
                           a.parts, uint32_t(spans), a.parts_row, n, a.target, a.labels, ignore_index, a.vocab, a.scale2,
                           lse2 + r, logp + r);
        e = status();
        if (e != SF_OK) return e;
    }
    return SF_OK;
}

int sf_logps_keep_grad(void* keep, size_t ld, size_t rows, size_t padded, size_t vocab, const void* parts,
                       const int64_t* labels, int64_t ignore_index, const float* lse2, const float* logp, int dtype,
                       const float* grad, size_t all_rows, float scale, float* row_weight, float* norm, int normalise,
                       sf_stream_t stream) {
    if (padded == 0) return SF_OK;
    if (rows > 0 && grad == nullptr) return SF_EINVAL;
    if (all_rows > 0 && (row_weight == nullptr || all_rows < rows || sizes_bad(all_rows, vocab) ||
                            (normalise && norm == nullptr)))
        return SF_EINVAL;
    if (keep == nullptr || parts == nullptr || labels == nullptr || lse2 == nullptr || logp == nullptr ||
        sizes_bad(padded, vocab) || padded < rows || ld < (vocab + kSpan - 1) / kSpan * kSpan || ld > (size_t(1) << 31))
        return SF_EINVAL;
    if (dtype != SF_DTYPE_BF16 && dtype != SF_DTYPE_F16) return SF_EDTYPE;
    if (misaligned(keep, 16) || misaligned(parts, 8) || ld % kSpan != 0) return SF_EALIGN;
    const uint32_t col_blocks = uint32_t((ld + kKeepColumns - 1) / kKeepColumns);
    const auto kernel = dtype == SF_DTYPE_BF16 ? logps_keep_grad_kernel<Bf16> : logps_keep_grad_kernel<F16>;
    const Weights weights = {grad, logp, labels, ignore_index, all_rows, uint32_t(vocab), scale, row_weight, norm,
                             dtype == SF_DTYPE_F16 ? 1.0f / kLift<F16> : 1.0f, normalise != 0};
    const uint64_t want = (all_rows + 4 * kGradThreads - 1) / (4 * kGradThreads);
    const uint32_t share = all_rows == 0 ? 0 : normalise ? 1 : uint32_t(want < 1024 ? want : 1024);
    return in_launches(uint64_t(padded) * col_blocks, [&](uint64_t first, uint32_t blocks) {
        const uint32_t others = first == 0 ? share : 0;
        hipLaunchKernelGGL(kernel, dim3(blocks + others), dim3(kGradThreads), 0, reinterpret_cast<hipStream_t>(stream),
                           static_cast<uint16_t*>(keep), uint64_t(ld), uint32_t(rows), uint32_t(vocab), col_blocks, first,
                           static_cast<const float2*>(parts), labels, ignore_index, lse2, logp, grad, weights, others);
    });
}

int sf_logps_rows(const float* logits, size_t ld, size_t rows, size_t vocab, const int64_t* labels,
                  int64_t ignore_index, float scale, float* lse, float* logp, sf_stream_t stream) {
    if (rows == 0) return SF_OK;
    if (logits == nullptr || labels == nullptr || lse == nullptr || logp == nullptr) return SF_EINVAL;
    if (sizes_bad(rows, vocab) || ld < vocab) return SF_EINVAL;
    if (misaligned(logits, 16) || ld % 4 != 0) return SF_EALIGN;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const uint32_t v = uint32_t(vocab);
    if (v <= 512) return launch_rows<16>(logits, ld, rows, v, labels, ignore_index, scale, lse, logp, st);
    if (v <= 4096) return launch_rows<64>(logits, ld, rows, v, labels, ignore_index, scale, lse, logp, st);
    if (v <= 16384) return launch_rows<256>(logits, ld, rows, v, labels, ignore_index, scale, lse, logp, st);
    return launch_rows<1024>(logits, ld, rows, v, labels, ignore_index, scale, lse, logp, st);
}

int sf_logps_hidden_grad(const void* d, size_t ld, size_t rows, const void* weight, size_t ldw, size_t vocab, size_t cols,
                         const float* row_weight, const float* norm, int dtype, void* out, sf_stream_t stream) {
    if (rows == 0) return SF_OK;
    if (d == nullptr || weight == nullptr || row_weight == nullptr || out == nullptr || sizes_bad(rows, vocab) ||
        cols == 0 || cols > (size_t(1) << 22) || ld < (vocab + 31) / 32 * 32 || ldw < cols)
        return SF_EINVAL;
    if (dtype != SF_DTYPE_BF16 && dtype != SF_DTYPE_F16) return SF_EDTYPE;
    if (cols % 8 != 0 || ld % 8 != 0 || ldw % 8 != 0 || misaligned(d, 16) || misaligned(weight, 16) || misaligned(out, 8))
        return SF_EALIGN;
    const uint64_t col_blocks = (cols + kHgColumns - 1) / kHgColumns;
    const uint64_t blocks = (uint64_t(rows) + kHgTokens - 1) / kHgTokens * col_blocks;
    if (blocks > kMaxLanes / (kHgWaves * 64)) return SF_EINVAL;
    const auto kernel = dtype == SF_DTYPE_BF16 ? logps_hidden_grad_kernel<Bf16> : logps_hidden_grad_kernel<F16>;
    hipLaunchKernelGGL(kernel, dim3(uint32_t(blocks)), dim3(kHgWaves * 64), 0, reinterpret_cast<hipStream_t>(stream),
                       static_cast<const uint16_t*>(d), uint64_t(ld), uint32_t(rows),
                       static_cast<const uint16_t*>(weight), uint64_t(ldw), uint32_t(vocab), uint32_t(cols),
                       uint32_t(col_blocks), row_weight, norm, static_cast<uint16_t*>(out));
    return status();
}

int sf_logps_weighted(const void* hidden, size_t ldh, size_t rows, size_t cols, const float* row_weight, int dtype,
                      void* out, sf_stream_t stream) {
    if (rows == 0) return SF_OK;
    if (hidden == nullptr || row_weight == nullptr || out == nullptr || sizes_bad(rows, cols) || ldh < cols)
        return SF_EINVAL;
    if (dtype != SF_DTYPE_BF16 && dtype != SF_DTYPE_F16) return SF_EDTYPE;
    if (cols % kGroup != 0 || ldh % kGroup != 0 || misaligned(hidden, 16) || misaligned(out, 16)) return SF_EALIGN;
    const auto kernel = dtype == SF_DTYPE_BF16 ? logps_weighted_kernel<Bf16> : logps_weighted_kernel<F16>;
    const uint64_t count = uint64_t(rows) * (cols / kGroup);
    return in_launches((count + kGradThreads - 1) / kGradThreads, [&](uint64_t first, uint32_t blocks) {
        hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kGradThreads), 0, reinterpret_cast<hipStream_t>(stream),
                           static_cast<const uint16_t*>(hidden), uint64_t(ldh), uint32_t(cols / kGroup), uint32_t(cols),
                           first, count, row_weight, static_cast<uint16_t*>(out));
    });
}

int sf_logps_hidden_product(const void* d, size_t ld, size_t rows, const void* weight, size_t ldw, size_t vocab,
                            size_t cols, int nparts, float* parts, int dtype, sf_stream_t stream) {
    return hidden_product(d, ld, rows, nullptr, weight, ldw, vocab, cols, nparts, parts, dtype, stream);
}

int sf_distill_hidden_product(const void* d, size_t ld, size_t rows, const int32_t* live, const void* weight, size_t ldw,
                              size_t vocab, size_t cols, int nparts, float* parts, int dtype, sf_stream_t stream) {
    if (live == nullptr || nparts > int(kMostLiveParts)) return SF_EINVAL;
    return hidden_product(d, ld, rows, live, weight, ldw, vocab, cols, nparts, parts, dtype, stream);
}

int sf_logps_weight_grad(const void* d, size_t ld, size_t tokens, size_t vocab, const void* hidden_t, size_t cols,
                         const float* norm, int dtype, void* out, sf_stream_t stream) {
    return weight_grad(d, ld, tokens, nullptr, vocab, hidden_t, cols, norm, dtype, out, stream);
}

int sf_distill_weight_grad(const void* d, size_t ld, size_t tokens, const int32_t* live, size_t vocab, const void* hidden_t,
                           size_t cols, const float* norm, int dtype, void* out, sf_stream_t stream) {
    if (live == nullptr) return SF_EINVAL;
    return weight_grad(d, ld, tokens, live, vocab, hidden_t, cols, norm, dtype, out, stream);
}

int sf_logps_weight(const float* grad, const float* logp, const int64_t* labels, int64_t ignore_index, size_t rows,
                    size_t vocab, float scale, float* weight, float* norm, sf_stream_t stream) {
    if (rows == 0 && norm == nullptr) return SF_OK;
    if (sizes_bad(rows, vocab) ||
        (rows > 0 && (grad == nullptr || logp == nullptr || labels == nullptr || weight == nullptr)))
        return SF_EINVAL;
    const uint64_t want = (rows + kWeightThreads - 1) / kWeightThreads;
    const uint32_t blocks = norm != nullptr ? 1 : uint32_t(want < 1024 ? want : 1024);
    const Weights a = {grad, logp, labels, ignore_index, rows, uint32_t(vocab), scale, weight, norm, 1.0f / kLift<F16>,
                       norm != nullptr};
    hipLaunchKernelGGL(logps_weight_kernel, dim3(blocks), dim3(kWeightThreads), 0, reinterpret_cast<hipStream_t>(stream), a);
    return status();
}

int sf_logps_grad(const float* logits, size_t ld, size_t rows, size_t vocab, const int64_t* labels,
                  int64_t ignore_index, float scale, const float* lse, const float* logp, const float* grad, void* dz,
                  int dtype, size_t ld_dz, sf_stream_t stream) {
    if (rows == 0) return SF_OK;
    if (logits == nullptr || labels == nullptr || lse == nullptr || logp == nullptr || grad == nullptr || dz == nullptr)
        return SF_EINVAL;
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
        return launch_grad<Out16<Bf16>>(logits, ld, rows, v, labels, ignore_index, scale, lse, logp, grad, dz, ld_dz, st);
    if (dtype == SF_DTYPE_F16)
        return launch_grad<Out16<F16>>(logits, ld, rows, v, labels, ignore_index, scale, lse, logp, grad, dz, ld_dz, st);
    return launch_grad<Out32>(logits, ld, rows, v, labels, ignore_index, scale, lse, logp, grad, dz, ld_dz, st);
}

}  // extern "C"
