// The product of the output unit's kernels with the softmax's sums in one, and
// what the gradients of log-probabilities and of distillation share.

#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/slidefsdp.h"
#include "sf_common.h"

namespace {

// What fp16 holds the kept exponentials and D times; D itself is within [-1, 1],
// but for the rounding of 1 - p_y, which could take fp16's product past its range.
template <typename Fmt>
constexpr float kLift = 1.0f;
template <>
constexpr float kLift<F16> = 0x1p14f;
template <typename Fmt>
__device__ __forceinline__ float lifted(float d) {   // d times kLift, not above 0
    if constexpr (kLift<Fmt> != 1.0f) return d < -kLift<Fmt> ? -kLift<Fmt> : d;
    return d;
}

// An exponential relative to its tile's maximum kept as 16 bits of -log2, 65535 for
// none: where no element of D is exact, a rounding of the exponential to bf16 before
// D's own shows (relative error of the gradients 2.6e-3, a rounding alone 1.7e-3).
// Steps of 2^-9 of an octave down to 2^-128 for bf16, within 2^-10.5 of itself, and
// of 2^-11 down to 2^-32 for fp16, whose D ends there too.
template <typename Fmt>
constexpr float kOctaves = 128.0f;
template <>
constexpr float kOctaves<F16> = 32.0f;
template <typename Fmt>
__device__ __forceinline__ uint32_t pack_log2(float a, float b) {   // a, b <= 0
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pknorm_u16(a * (-1.0f / kOctaves<Fmt>), b * (-1.0f / kOctaves<Fmt>)));
}
// 2^(more - what is kept); 0 of none, whatever more is: the columns that pad a last tile whose
// words are all picked are relative to no maximum, and more is above 0 where the other words are far below.
template <typename Fmt>
__device__ __forceinline__ float exp2_kept(uint32_t u, float more) {
    const float e = __builtin_amdgcn_exp2f(fmaf(float(u), -kOctaves<Fmt> / 65535.0f, more));
    return u == 65535 ? 0.0f : e;
}

// ---------------------------------------------------------------------
// The product with the softmax's sums.  A workgroup has a tile of 256 words
// by kBT tokens, a wave kFV x kFT products of 16 x 16 (words are the rows of
// the product: a lane then holds 4 kFV words of each of its kFT tokens, and a
// token's sums take two exchanges between lanes).
//
// The operands go from memory to LDS without passing registers, 64 terms of
// the sum at a time in two buffers, 16-byte chunk c of row r at c ^ (r % 8) so
// that a wave's reads of a column of chunks touch every bank.  The products of
// one half (32 terms) run while the operands of the next are read from LDS;
// one barrier for each 64 terms, at which the next buffer has arrived (it had
// the time of 64 terms) and this one is free.
//
// Workgroups that run side by side on an XCD take neighbouring tiles, up to 8
// of tokens by 4 of words: what they read is in its L2 once.
// ---------------------------------------------------------------------
constexpr int kSpan = SF_LOGPS_SPAN;   // words of a tile
constexpr int kTerms = 64;             // of a buffer
constexpr int kRowBytes = kTerms * 2;
constexpr int kGroupT = 8;             // tiles of tokens that run side by side

struct Tiles {
    const uint16_t* weight;   // [vocab, 64 steps], ldw
    const uint16_t* hidden;   // [tokens, 64 steps], ldh
    uint32_t ldw, ldh, vocab, tokens, steps;
    const int64_t* labels;
    const int32_t* order;     // [tokens + 1] the rows with a label and their number, or null: all rows
    float scale2;             // scale * log2(e)
    float2* parts;            // [tiles of words, parts_row] maximum in base 2 (kPick: as it is) and sum
    uint64_t parts_row;       // tokens of the whole call, of which these are some
    float* target;            // [tokens] the label's product, unscaled
    uint16_t* keep;           // [tokens, ld_keep] or null
    uint64_t ld_keep;
    // Where words of each token are picked out, in place of labels and target:
    const int32_t* words;     // [tokens, picks] each token's, rising
    const uint8_t* starts;    // [tokens, tiles of words + 1] its first of each tile
    float* picked;            // [tokens, picks] their products, unscaled
    uint32_t picks;
    bool close;               // keep's rows in the order of `order`, without gaps
};

// The rows that have(i), in their order, and behind `rows` of them their number.
// The product skips the others, prompts above all: their share of its time for
// one launch, 5 us at 8190 rows.  One workgroup, each lane a run of rows.
constexpr int kOrderThreads = 1024;
template <typename Have>
__global__ __launch_bounds__(kOrderThreads) void logps_order_kernel(const Have have, uint32_t rows,
                                                                    int32_t* __restrict__ order) {
    __shared__ uint32_t waves[kOrderThreads / 64];
    const uint32_t each = (rows + kOrderThreads - 1) / kOrderThreads;
    const uint32_t from = min(threadIdx.x * each, rows), to = min(from + each, rows);
    uint32_t mine = 0;
    for (uint32_t i = from; i < to; ++i) mine += have(i);
    uint32_t before = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t below = __shfl_up(before, d);
        if ((threadIdx.x & 63) >= uint32_t(d)) before += below;
    }
    if ((threadIdx.x & 63) == 63) waves[threadIdx.x >> 6] = before;
    before -= mine;
    __syncthreads();
    for (uint32_t w = 0; w < (threadIdx.x >> 6); ++w) before += waves[w];
    for (uint32_t i = from; i < to; ++i)
        if (have(i)) order[before++] = int32_t(i);
    if (threadIdx.x == kOrderThreads - 1) order[rows] = int32_t(before);
}

// Parts of the hidden gradient's sum over `steps` of 64 words, at most `most`, where the device
// alone knows the rows: by rounds of 256 compute units that the tiles of 256 x 256 take, and by
// what adding a part up costs, as much as 20 steps of its tiles.  Product and sum in us, the
// host's parts for all rows | these, a fifth of the rows masked: 4092 x 4096 x 128256 2923 (1) |
// 2849 (6), 8190 x 5120 x 152064 9728 (2) | 8870 (6); a step with half of them masked 6927 | 5499
// and 16894 | 15796, 16384 x 2048 x 50257 5995 | 4767.  Whole numbers: the product and the sum
// come to the same.  All lanes of a wave call it, each weighs a number of its own.
constexpr uint32_t kMostLiveParts = 16;
__device__ __forceinline__ uint32_t parts_of_rows(uint32_t rows, uint32_t cols, uint32_t steps, uint32_t most) {
    const uint32_t p = (threadIdx.x & (kMostLiveParts - 1)) + 1, each = (steps + p - 1) / p;
    const uint64_t tiles = uint64_t((rows + 255) / 256) * ((cols + 255) / 256);
    uint64_t least = ((tiles * p + 255) / 256 * each * 256 + tiles * p * 20) << 5 | p;
    if (p > most || (steps + each - 1) / each != p) least = ~uint64_t(0) << 5 | 1;   // or a part would be empty
#pragma unroll
    for (int d = 1; d < int(kMostLiveParts); d <<= 1) least = min(least, uint64_t(__shfl_xor(least, d)));
    return uint32_t(least) & 31;
}

// Interleaves what a half's products run beside: kLoads copies into LDS, then
// kReads reads of it, two products each; all else after.
template <int kReads, int kMul, int kLoads>
__device__ __forceinline__ void interleave() {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x010, 1, 0);   // memory
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);   // product
    }
#pragma unroll
    for (int i = 0; i < kReads; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);   // LDS read
        __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, kMul, 0);
}

// kWV x kWT waves of words and of tokens.  kDeep buffers of 64 terms each: all
// but one are on their way while one is used.  kOrder: tokens in the order of
// a.order, otherwise all of them.  kPick: a token's words leave the tile for
// a.picked, before its maximum and its sum, which are then those of all others, and
// kept are logarithms (pack_log2).  Its maximum stays unscaled and is subtracted before
// the scale: differences hold at low temperatures, however large the logits over them
// are.  With 64 words a token and a fifth of the tokens left out 2,810-2,870 us at 4092 x
// 4096 x 128256, 8,250-8,580 at 8190 x 5120 x 152064 (by the box), 1.2 PFLOP/s of the
// rows that count; with one label picked by its index 2,832 and 8,394.
template <typename Fmt, int kWV, int kWT, int kFV, int kFT, int kDeep, bool kKeep, bool kOrder, bool kPick>
__global__ __launch_bounds__(kWV * kWT * 64, 2) void logps_tiles_kernel(const Tiles a) {
    constexpr int kWaves = kWV * kWT, kBV = kWV * kFV * 16, kBT = kWT * kFT * 16;
    static_assert(kBV == kSpan, "a tile is one span of words");
    constexpr int kBuffer = (kBV + kBT) * kRowBytes;
    constexpr int kLV = kBV / 8 / kWaves, kLT = kBT / 8 / kWaves;   // a wave copies 8 rows at once
    static_assert(kLV * 8 * kWaves == kBV && kLT * 8 * kWaves == kBT, "rows divide among the waves");
    // The end exchanges maxima and sums between the waves and turns each wave's 16
    // tokens of kept words around, over the buffers.
    constexpr int kTurnRow = kFV * 32;   // bytes of a token's words of a wave
    static_assert(kWaves * 16 * kTurnRow <= kDeep * kBuffer && kWV * kBT * 4 <= kDeep * kBuffer, "the buffers hold it");
    // Where LDS has room for it and a compute unit only one workgroup: each token's
    // row and label (-1: none inside the vocabulary), which the end would otherwise
    // wait for.
    constexpr int kLds = 160 * 1024;
    constexpr bool kNoted = 2 * kDeep * kBuffer > kLds && kDeep * kBuffer + kBT * 8 <= kLds;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[kDeep * kBuffer + (kNoted ? kBT * 8 : 0)];
    int32_t* const noted_row = reinterpret_cast<int32_t*>(lds + kDeep * kBuffer);
    int32_t* const noted_label = noted_row + kBT;

    const uint32_t lane = threadIdx.x & 63, l16 = lane & 15, quad = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t wv = wave / kWT, wt = wave % kWT, wv0 = wv * kFV * 16, wt0 = wt * kFT * 16;

    // Workgroups go to the XCDs in turn: each XCD has a contiguous run of tiles;
    // those that no token needs end here.
    const uint32_t count = kOrder ? uint32_t(a.order[a.tokens]) : a.tokens;
    const uint32_t tiles_v = (a.vocab + kBV - 1) / kBV, tiles_t = (count + kBT - 1) / kBT, tiles = tiles_v * tiles_t;
    const uint32_t xcd = blockIdx.x % 8, each = tiles / 8, more = tiles % 8;
    if (blockIdx.x / 8 >= each + (xcd < more)) return;
    const uint32_t id = xcd * each + min(xcd, more) + blockIdx.x / 8;
    const auto row_of = [&](uint32_t token) {   // past the last one: the last one's
        token = min(token, count - 1);
        return kOrder ? uint32_t(a.order[token]) : token;
    };
    const uint32_t first_t = id / (kGroupT * tiles_v) * kGroupT, group_t = min(uint32_t(kGroupT), tiles_t - first_t);
    const uint32_t in = id - first_t * tiles_v;
    const uint32_t v0 = in / group_t * kBV, t0 = (first_t + in % group_t) * kBT;
    const auto label_of = [&](uint32_t token, uint32_t row) {   // kPick: its first word here, and behind 8 bits its end
        if constexpr (kPick) {
            if (token >= count) return 0;
            const uint8_t* s = a.starts + uint64_t(row) * (tiles_v + 1) + v0 / kBV;
            return int32_t(s[0] | s[1] << 8);
        }
        const int64_t y = a.labels[row];
        return token < count && y >= 0 && y < int64_t(a.vocab) ? int32_t(y) : -1;
    };

    const uint8_t* gv = reinterpret_cast<const uint8_t*>(a.weight + uint64_t(v0) * a.ldw);
    const uint32_t t_base = kOrder ? 0 : t0;
    const uint8_t* gt = reinterpret_cast<const uint8_t*>(a.hidden + uint64_t(t_base) * a.ldh);
    // Rows past the last are the last one again: their results are dropped below.
    uint32_t off[kLV + kLT];
    const uint32_t chunk = ((lane & 7) ^ (lane >> 3)) * 16;
#pragma unroll
    for (int j = 0; j < kLV; ++j)
        off[j] = min((j * kWaves + wave) * 8 + (lane >> 3), a.vocab - 1 - v0) * (a.ldw * 2) + chunk;
#pragma unroll
    for (int j = 0; j < kLT; ++j)
        off[kLV + j] = (row_of(t0 + (j * kWaves + wave) * 8 + (lane >> 3)) - t_base) * (a.ldh * 2) + chunk;
    typedef __attribute__((address_space(3))) uint8_t Lds;
    typedef const __attribute__((address_space(1))) uint8_t Global;
    const auto copy = [&](uint32_t step, uint32_t buf) {
        uint8_t* to = lds + buf * kBuffer + wave * 1024;
#pragma unroll
        for (int j = 0; j < kLV; ++j)
            __builtin_amdgcn_global_load_lds((Global*)(gv + step * kRowBytes + off[j]),
                                             (Lds*)(to + j * kWaves * 1024), 16, 0, 0);
#pragma unroll
        for (int j = 0; j < kLT; ++j)
            __builtin_amdgcn_global_load_lds((Global*)(gt + step * kRowBytes + off[kLV + j]),
                                             (Lds*)(to + kBV * kRowBytes + j * kWaves * 1024), 16, 0, 0);
    };
    const uint32_t at = (quad ^ (l16 & 7)) * 16;
    const uint32_t at_v = (wv * kFV * 16 + l16) * kRowBytes, at_t = (kBV + wt * kFT * 16 + l16) * kRowBytes;
    u32x4 x[2][kFV], y[2][kFT];
    const auto read = [&](uint32_t buf, int half) {
        const uint8_t* from = lds + buf * kBuffer + (at ^ (half * 64));
#pragma unroll
        for (int i = 0; i < kFV; ++i) x[half][i] = *reinterpret_cast<const u32x4*>(from + at_v + i * 16 * kRowBytes);
#pragma unroll
        for (int j = 0; j < kFT; ++j) y[half][j] = *reinterpret_cast<const u32x4*>(from + at_t + j * 16 * kRowBytes);
    };
    f32x4 acc[kFV][kFT];
    const auto multiply = [&](int half) {
#pragma unroll
        for (int i = 0; i < kFV; ++i)
#pragma unroll
            for (int j = 0; j < kFT; ++j) acc[i][j] = mfma(Fmt{}, x[half][i], y[half][j], acc[i][j]);
    };
    // Every wave's LDS reads are done, and its copies but those of the last `ahead`
    // buffers; nothing moves across.
    const auto meet = [](auto ahead) {
        constexpr uint32_t kLeft = decltype(ahead)::value * (kLV + kLT);
        static_assert(kLeft < 64, "what the counter holds");
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0x0070 | (kLeft & 15) | kLeft >> 4 << 14);
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    // kMore: there are buffers left to copy
    const auto step = [&](uint32_t s, auto kMore) {
        read(s % kDeep, 1);
        multiply(0);
        interleave<kFV + kFT, kFV * kFT, 0>();
        if constexpr (decltype(kMore)::value) {
            meet(std::integral_constant<int, kDeep - 2>{});
            copy(s + kDeep, s % kDeep);
        } else {
            meet(std::integral_constant<int, 0>{});
        }
        read((s + 1) % kDeep, 0);
        multiply(1);
        interleave<kFV + kFT, kFV * kFT, decltype(kMore)::value ? kLV + kLT : 0>();
        __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (int i = 0; i < kFV; ++i)
#pragma unroll
        for (int j = 0; j < kFT; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int d = 0; d < kDeep; ++d)
        if (uint32_t(d) < a.steps) copy(d, d);
    if (kNoted && threadIdx.x < kBT) {
        const uint32_t token = t0 + threadIdx.x, row = row_of(token);
        noted_row[threadIdx.x] = int32_t(row);
        noted_label[threadIdx.x] = label_of(token, row);
    }
    // The note above waits for its own loads: the counter is at 0 with them, so the
    // first buffer needs no other rule.
    meet(std::integral_constant<int, 0>{});
    read(0, 0);
    uint32_t s = 0;
    for (; s + kDeep < a.steps; ++s) step(s, std::true_type{});
    while (s + 1 < a.steps) step(s++, std::false_type{});
    read(s % kDeep, 1);
    multiply(0);
    interleave<kFV + kFT, kFV * kFT, 0>();
    meet(std::integral_constant<int, 0>{});   // the buffers are not read again
    multiply(1);
    uint32_t row[kFT];
    int32_t label[kFT];   // as an index from this lane's first word
#pragma unroll
    for (int j = 0; j < kFT; ++j) {
        const uint32_t t = wt0 + j * 16 + l16;
        row[j] = kNoted ? uint32_t(noted_row[t]) : row_of(t0 + t);
        if constexpr (kPick) continue;
        label[j] = kNoted ? noted_label[t] : label_of(t0 + t, row[j]);
        if (label[j] >= 0) label[j] -= int32_t(v0 + wv0 + quad * 4);
    }

    if (v0 + kBV > a.vocab) {
#pragma unroll
        for (int i = 0; i < kFV; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (v0 + wv0 + i * 16 + quad * 4 + r >= a.vocab)
#pragma unroll
                    for (int j = 0; j < kFT; ++j) acc[i][j][r] = -__builtin_inff();
    }
    if constexpr (kPick) {
        // A token's words among these 256 as bits, behind them the place of the first; a
        // token has few here, most have none (64 of 128256 words: 0.13 a tile).
        constexpr int kMark = kSpan / 32 + 1;
        static_assert(kBT <= kWaves * 64 && kWV * kBT * 4 + kBT * kMark * 4 <= kDeep * kBuffer, "one lane a token");
        uint32_t* const marks = reinterpret_cast<uint32_t*>(lds + kWV * kBT * 4);
        if (threadIdx.x < kBT) {
            const uint32_t token = t0 + threadIdx.x, at = kNoted ? uint32_t(noted_row[threadIdx.x]) : row_of(token);
            const uint32_t range = uint32_t(kNoted ? noted_label[threadIdx.x] : label_of(token, at));
            uint32_t* const mine = marks + threadIdx.x * kMark;
#pragma unroll
            for (int b = 0; b < kMark - 1; ++b) mine[b] = 0;
            mine[kMark - 1] = range & 255;
            for (uint32_t k = range & 255; k < range >> 8; ++k) {
                const uint32_t w = uint32_t(a.words[uint64_t(at) * a.picks + k]) - v0;
                mine[w / 32] |= 1u << w % 32;
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kFT; ++j) {
            const uint32_t* const of = marks + (wt0 + j * 16 + l16) * kMark;
            uint32_t bits[kFV / 2], any = 0;
#pragma unroll
            for (int b = 0; b < kFV / 2; ++b) any |= bits[b] = of[wv0 / 32 + b];
            if (any == 0) continue;
            uint32_t at = of[kMark - 1];
            for (uint32_t b = 0; b < wv0 / 32; ++b) at += __popc(of[b]);
            float* const to = a.picked + uint64_t(row[j]) * a.picks;
#pragma unroll
            for (int i = 0; i < kFV; ++i) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const uint32_t bit = i % 2 * 16 + quad * 4 + r;
                    if (bits[i / 2] >> bit & 1) {
                        to[at + __popc(bits[i / 2] & ((1u << bit) - 1))] = acc[i][j][r];
                        acc[i][j][r] = -__builtin_inff();
                    }
                }
                if (i % 2) at += __popc(bits[i / 2]);
            }
        }
    }
    float* const shared = reinterpret_cast<float*>(lds);   // [kWV][kBT]
    float top[kFT], sum[kFT];
#pragma unroll
    for (int j = 0; j < kFT; ++j) {
        float m = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < kFV; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) m = fmaxf(m, acc[i][j][r]);
        m = fmaxf(m, __shfl_xor(m, 16));
        m = fmaxf(m, __shfl_xor(m, 32));
        if (quad == 0) shared[wv * kBT + wt0 + j * 16 + l16] = m;
        // the label's product, by the one lane that has it
        if constexpr (kPick) continue;
        if (uint32_t(label[j]) < uint32_t(kFV * 16) && (label[j] & 15) < 4) {
            float z = 0.0f;
#pragma unroll
            for (int i = 0; i < kFV; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (label[j] == i * 16 + r) z = acc[i][j][r];
            a.target[row[j]] = z;
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kFT; ++j) {
        const uint32_t t = wt0 + j * 16 + l16;
        float m = shared[t];
#pragma unroll
        for (int w = 1; w < kWV; ++w) m = fmaxf(m, shared[w * kBT + t]);
        top[j] = kPick ? m : m * a.scale2;
    }
    __syncthreads();   // read by all before it is overwritten
    uint8_t* const turn = lds + wave * 16 * kTurnRow;
#pragma unroll
    for (int j = 0; j < kFT; ++j) {
        // exp2(scale2 x - base(top)): the product is not rounded before the difference, or (kPick)
        // exp2(scale2 (x - base(top)))
        const float c = base(top[j]);
        sum[j] = 0.0f;
#pragma unroll
        for (int i = 0; i < kFV; ++i) {
            f32x4 t, e;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                t[r] = kPick ? (acc[i][j][r] - c) * a.scale2 : fmaf(acc[i][j][r], a.scale2, -c);
                e[r] = __builtin_amdgcn_exp2f(t[r]);
                sum[j] += e[r];
            }
            if constexpr (kKeep) {
                const uint32_t to = ((i * 2 + (quad >> 1)) ^ (l16 & (kFV * 2 - 1))) * 16 + (quad & 1) * 8;
                *reinterpret_cast<u32x2*>(turn + l16 * kTurnRow + to) =
                    kPick ? u32x2{pack_log2<Fmt>(t[0], t[1]), pack_log2<Fmt>(t[2], t[3])}
                          : u32x2{Fmt::pack(e[0] * kLift<Fmt>, e[1] * kLift<Fmt>), Fmt::pack(e[2] * kLift<Fmt>, e[3] * kLift<Fmt>)};
            }
        }
        sum[j] += __shfl_xor(sum[j], 16);
        sum[j] += __shfl_xor(sum[j], 32);
        if constexpr (kKeep) {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            constexpr int kAcross = kTurnRow / 16, kRows = 64 / kAcross;   // lanes of a row, rows at once
#pragma unroll
            for (int k = 0; k < 16 / kRows; ++k) {
                const uint32_t r = k * kRows + lane / kAcross, c16 = lane % kAcross;
                const u32x4 v = *reinterpret_cast<const u32x4*>(turn + r * kTurnRow + (c16 ^ (r & (kFV * 2 - 1))) * 16);
                const uint32_t from = __shfl(row[j], r);   // of the lane that has this token
                const uint32_t to = kPick && a.close ? t0 + wt0 + j * 16 + r : from;
                if (t0 + wt0 + j * 16 + r < count)
                    *reinterpret_cast<u32x4*>(a.keep + to * a.ld_keep + v0 + wv0 + c16 * 8) = v;
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
    }
    if constexpr (kKeep) __syncthreads();
    if (wv > 0 && quad == 0)
#pragma unroll
        for (int j = 0; j < kFT; ++j) shared[wv * kBT + wt0 + j * 16 + l16] = sum[j];
    __syncthreads();
    if (wv == 0 && quad == 0)
#pragma unroll
        for (int j = 0; j < kFT; ++j) {
            const uint32_t t = wt0 + j * 16 + l16;
#pragma unroll
            for (int w = 1; w < kWV; ++w) sum[j] += shared[w * kBT + t];
            if (t0 + t < count) a.parts[uint64_t(v0 / kSpan) * a.parts_row + row[j]] = float2{top[j], sum[j]};
        }
}

template <typename Fmt, bool kPick, int kWV, int kWT, int kFV, int kFT, int kDeep>
int launch_tiles(const Tiles& a, hipStream_t st) {
    constexpr uint32_t kBT = kWT * kFT * 16;
    const uint64_t tiles = uint64_t((a.vocab + kSpan - 1) / kSpan) * ((a.tokens + kBT - 1) / kBT);
    const auto all = a.keep != nullptr ? logps_tiles_kernel<Fmt, kWV, kWT, kFV, kFT, kDeep, true, false, kPick>
                                       : logps_tiles_kernel<Fmt, kWV, kWT, kFV, kFT, kDeep, false, false, kPick>;
    const auto some = a.keep != nullptr ? logps_tiles_kernel<Fmt, kWV, kWT, kFV, kFT, kDeep, true, true, kPick>
                                        : logps_tiles_kernel<Fmt, kWV, kWT, kFV, kFT, kDeep, false, true, kPick>;
    const auto kernel = a.order != nullptr ? some : all;
    hipLaunchKernelGGL(kernel, dim3(uint32_t(tiles)), dim3(kWV * kWT * 64), 0, st, a);
    return status();
}

// The tile for a call: tokens of a tile, and the time of a round of them over
// the chip (256 tiles of 256 or 128 tokens, 512 of the smaller ones, of which a
// compute unit holds two; `half`: where there is at most one for each unit), in
// that of a round of the largest.  Small sums (`brief`, under 2048 terms) spend
// more of it at the ends of their tiles.  Measured, us, 256 | 128 | 64 | 32
// tokens a tile: 128256 words x 4096 terms and 64 tokens 220 | 178 | 171 | 203,
// 128 tokens 218 | 204 | 217 | 331, 256 tokens 230 | 349 | 356 | 586, 1023
// tokens 799 | 1207 | 1166 | 2028; 777 tokens x 1024, 50257 words 109 | 101 |
// 98 | 168, 32000 words 58 | 68 | 65 | 113; 300 x 2560 x 8192 51 | 36 | 35 | 41,
// 126 x 2048 x 16384 42 | 29 | 28 | 22, 8000 x 1024 x 1000 27 | 20 | 22 | 30.
//
// Buffers: what fits, but where two workgroups are to share a compute unit's LDS.
// 128 tokens with 3 against 2: 200 x 4096 x 32000 64 against 76 us, 64 x 4096 x
// 128256 178 against 200, at the worst (1000 x 1024 x 2000) 17.9 against 17.2.
// 32 tokens with 4 against 2, at one tile a unit: 64 x 4096 x 32000 47 against 59
// us, 126 x 2048 x 16384 22 against 26, 126 x 512 x 4096 (a weight that stays in
// L2) 8.8 against 8.4.  With two tiles a unit, 4 buffers cost what the second
// tile gives: 200 x 4096 x 32000 138 against 113 us.
struct TileKind {
    uint32_t tokens, slots, lanes;
    float round, half, brief, brief_half;
};
constexpr TileKind kTileKinds[] = {
    {256, 256, 512, 1.00f, 1.00f, 1.00f, 1.00f},
    {128, 256, 512, 0.75f, 0.68f, 0.60f, 0.60f},
    {64, 512, 256, 0.76f, 0.66f, 0.60f, 0.57f},
    {32, 512, 256, 0.78f, 0.53f, 0.60f, 0.50f},
};

template <typename Fmt, bool kPick>
int dispatch_tiles(const Tiles& a, hipStream_t st) {
    const uint64_t spans = (a.vocab + kSpan - 1) / kSpan;
    const bool brief = a.steps * kTerms < 2048;
    uint32_t best = 0;
    bool alone = false;
    float least = 0.0f;
    for (const TileKind& k : kTileKinds) {
        const uint64_t tiles = spans * ((a.tokens + k.tokens - 1) / k.tokens);
        if (tiles > kMaxLanes / k.lanes) continue;   // never of the first kind
        const float one = tiles <= 256 ? (brief ? k.brief_half : k.half) : brief ? k.brief : k.round;
        const float time = one * float((tiles + k.slots - 1) / k.slots);
        if (best == 0 || time < least) best = k.tokens, least = time, alone = tiles <= 256;
    }
    switch (best) {
        case 32: return alone ? launch_tiles<Fmt, kPick, 4, 1, 4, 2, 4>(a, st) : launch_tiles<Fmt, kPick, 4, 1, 4, 2, 2>(a, st);
        case 64: return launch_tiles<Fmt, kPick, 4, 1, 4, 4, 2>(a, st);
        case 128: return launch_tiles<Fmt, kPick, 4, 2, 4, 4, 3>(a, st);
        default: return launch_tiles<Fmt, kPick, 2, 4, 8, 4, 2>(a, st);
    }
}

// Rows' weights: what multiplies each row of D in the products, or a hidden row before them.
// The share of workgroup `block` of `blocks`; one alone where they are normalised.
// a(i): row i's.
template <int kT, typename Weights>
__device__ __forceinline__ void row_weights(const Weights& a, uint64_t block, uint64_t blocks) {
    float by = 1.0f, back = 1.0f;
    if (a.normalise) {
        __shared__ float waves[kT / 64];
        float m = 0.0f;
        for (uint64_t i = threadIdx.x; i < a.n; i += kT) {
            const float w = fabsf(a(i));
            if (__builtin_isfinite(w)) m = fmaxf(m, w);
        }
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
        if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = m;
        __syncthreads();
        m = waves[0];
        for (int w = 1; w < kT / 64; ++w) m = fmaxf(m, waves[w]);
        // within what both the factor and its inverse can be
        const int e = m > 0.0f ? min(max(ilogbf(m) + 1, -100), 100) : 0;
        by = ldexpf(1.0f, -e), back = ldexpf(1.0f, e);
    }
    for (uint64_t i = block * kT + threadIdx.x; i < a.n; i += blocks * kT) a.weight[i] = a(i) * by;
    if (a.norm != nullptr && block == 0 && threadIdx.x == 0) a.norm[0] = back * a.unlift, a.norm[1] = 1.0f;
}

}  // namespace
