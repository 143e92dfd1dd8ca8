// The largest log-probabilities of rows of logits, and one token drawn from each
// row after temperature, top-k, top-p and min-p, for MI355X (gfx950).
//
// Words are ordered by falling logit, the first of equals first.  With w_j =
// exp((x_j - max) / T) a row keeps a prefix of that order: the first top_k; of
// those the words with less than top_p of their mass before them; of those the
// words with w_j >= min_p.  The word drawn is the first kept one, by its index,
// whose running mass exceeds u times the kept mass: no sort of the vocabulary.
// Which word that is hangs on sums of up to 2^30 terms, so the masses that decide it are
// 64-bit.  (The mass of all words of a row that goes by lists is for its log-probability
// alone: a lane's 64 are summed in fp32.)
//
// Two launches.  rows_parts_kernel cuts rows into parts of up to 2048 16-byte
// vectors, which a workgroup holds in registers, and leaves of each its maximum,
// its mass relative to that, and what the row's border will need: the words that
// may be among the k largest of it, or a histogram of its masses.  The chip is
// filled by parts, whatever the rows.  A workgroup for each row then joins its
// parts.  The k largest are picked from the parts' lists by one wave, without a
// barrier.  A border by mass lies in one bin of the joined histograms, whose few
// hundred words are read and binned again; the histograms also say how much of its
// mass each part keeps, so that the word is looked for in one part alone.  Rows
// whose words tie or spread so that this does not do (more candidates than their
// lists hold, a border below the histogram) find their border by radix passes
// over the row.
//
// Sums of masses are added in a fixed order in fp64, or in whole numbers where the
// order is not fixed: results are the same from call to call.
//
// C ABI: include/slidefsdp.h.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/slidefsdp.h"
#include "sf_common.h"

namespace {

constexpr uint32_t kMost = SF_TOP_MOST;   // words that the parts' lists are made for
constexpr uint32_t kPartLanes = 256;
constexpr uint32_t kPartVectors = 8;      // of a lane
// Of a part's histogram, T / kBinsOfT of logit each: down to e^-32 of the largest weight.  A
// vocabulary's many small ones are beyond e^-16 of a sure word and still a thousandth of the
// mass together.
constexpr uint32_t kBins = 512;
constexpr float kBinsOfT = 16.0f;
constexpr uint32_t kList = kBins + kBins / 4;   // candidates of a part, of a row's only part twice as many
constexpr uint32_t kSubBins = 1024;       // of a bin
constexpr uint32_t kDigit = 8;            // bits of a radix pass
constexpr uint32_t kMostParts = 64;       // of a row that goes by histograms
constexpr float kNegInf = -__builtin_inff();

// fp32 rows beside the 16-bit formats: what a 16-byte vector holds.
struct F32 {};
template <typename E>
constexpr uint32_t kOf = std::is_same_v<E, F32> ? 4 : 8;
template <typename E>
using Item = std::conditional_t<std::is_same_v<E, F32>, uint32_t, uint16_t>;

template <typename E>
__device__ __forceinline__ float item(u32x4 v, uint32_t i) {
    if constexpr (std::is_same_v<E, F32>) return __uint_as_float(v[i]);
    else return i % 2 ? E::hi(v[i / 2]) : E::lo(v[i / 2]);
}

template <typename E>
__device__ __forceinline__ float item_at(u32x4 v, uint32_t i) {
    constexpr uint32_t kA = std::is_same_v<E, F32> ? 1 : 2;   // of a word
    uint32_t word = v[0];
#pragma unroll
    for (uint32_t w = 1; w < 4; ++w) word = i / kA == w ? v[w] : word;
    return item<E>(u32x4{word, 0, 0, 0}, kA == 1 ? 0 : i % 2);
}

// Order-preserving words of floats; -0 as 0.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float float_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}
// A word's place in its row's order: larger is earlier, all are different.
__device__ __forceinline__ uint64_t place_of(float x, uint32_t index) {
    return uint64_t(key_of(x)) << 32 | uint32_t(~index);
}
__device__ __forceinline__ float logit_of(uint64_t place) { return float_of(uint32_t(place >> 32)); }
__device__ __forceinline__ uint32_t index_of(uint64_t place) { return ~uint32_t(place); }

// 2^y for y <= 0 or so, 0 of -inf: 2^n times the series of e^(f ln 2) to its 10th power, off
// by 2^-42 of itself.
constexpr int kPowers = 10;
struct Series {
    double c[kPowers + 1];
    constexpr Series() : c() {
        c[0] = 1.0;
        for (int i = 1; i <= kPowers; ++i) c[i] = c[i - 1] * 0.69314718055994530941723212145818 / i;
    }
};
__constant__ constexpr Series kSeries{};
__device__ __forceinline__ double exp2_wide(double y) {
    y = fmax(y, -1100.0);
    const double n = rint(y), f = y - n;
    double p = kSeries.c[kPowers];
#pragma unroll
    for (int i = kPowers - 1; i >= 0; --i) p = fma(p, f, kSeries.c[i]);
    return ldexp(p, int(n));
}
// A logit's weight, exp((x - from) / T) as 2^(c (x - from)); 0 of -inf.
struct Weigh {
    double c, from;
    __device__ Weigh(double c_, float from_) : c(c_), from(from_) {}
    __device__ double operator()(float x) const {
        return exp2_wide((double(x) - from) * c);
    }
};

template <typename E>
__device__ __forceinline__ u32x4 nothing() {
    const uint32_t w = std::is_same_v<E, F32> ? 0xFF800000u : std::is_same_v<E, Bf16> ? Bf16::kNegInf2 : F16::kNegInf2;
    return u32x4{w, w, w, w};
}

// A row's vectors: whole 16-byte ones but for its first and its last, which may lie
// partly outside and are read by elements, -inf where they are not the row's.
template <typename E>
struct Row {
    const Item<E>* x;
    uint32_t vocab, shift, vectors;   // the row begins `shift` elements into vector 0
    uint32_t first, end;              // whole vectors
    __device__ Row(const void* logits, uint64_t ld, uint64_t row, uint32_t vocab_) : vocab(vocab_) {
        x = static_cast<const Item<E>*>(logits) + row * ld;
        shift = uint32_t(reinterpret_cast<uintptr_t>(x) % 16) / sizeof(Item<E>);
        vectors = (vocab + shift + kOf<E> - 1) / kOf<E>;
        first = shift > 0 ? 1 : 0, end = max((vocab + shift) / kOf<E>, first);
    }
    // kN vectors, that(i) each: all whole ones on their way at once, without a branch between
    // them, which would wait; from `vectors` on -inf.  Vector 0 is the first, if any.
    template <uint32_t kN, typename That>
    __device__ __forceinline__ void load(u32x4 (&r)[kN], That that) const {
        if (end > first) {
#pragma unroll
            for (uint32_t i = 0; i < kN; ++i) {
                const uint32_t v = that(i), u = min(max(v, first), end - 1);
                r[i] = reinterpret_cast<const u32x4*>(x - shift)[u];
            }
#pragma unroll
            for (uint32_t i = 0; i < kN; ++i)
                if (that(i) != min(max(that(i), first), end - 1)) r[i] = nothing<E>();
        } else {
#pragma unroll
            for (uint32_t i = 0; i < kN; ++i) r[i] = nothing<E>();
        }
        if (first > 0 && that(0) == 0) r[0] = edge(0);
        if (end < vectors) {
            bool has = false;
#pragma unroll
            for (uint32_t i = 0; i < kN; ++i) has |= that(i) == vectors - 1;
            if (has) {
                const u32x4 last = edge(vectors - 1);
#pragma unroll
                for (uint32_t i = 0; i < kN; ++i)
                    if (that(i) == vectors - 1) r[i] = last;
            }
        }
    }
    __device__ u32x4 edge(uint32_t v) const {
        const int64_t at = int64_t(v) * kOf<E> - shift;
        u32x4 r;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            if constexpr (std::is_same_v<E, F32>) {
                r[i] = uint64_t(at + i) < vocab ? x[at + i] : 0xFF800000u;
            } else {
                const uint32_t lo = uint64_t(at + 2 * i) < vocab ? x[at + 2 * i] : E::kNegInf;
                const uint32_t hi = uint64_t(at + 2 * i + 1) < vocab ? x[at + 2 * i + 1] : E::kNegInf;
                r[i] = lo | hi << 16;
            }
        }
        return r;
    }
    __device__ float at(uint32_t index) const {
        if constexpr (std::is_same_v<E, F32>) return __uint_as_float(x[index]);
        else return E::lo(x[index]);
    }
    __device__ uint32_t index(uint32_t v, uint32_t i) const { return v * kOf<E> + i - shift; }
};

// What a part leaves.
struct Part {
    float m;          // its largest logit
    uint32_t count;   // candidates, also those that its list does not hold
    double sum;       // of exp((x - m) / T); NaN with one among its logits
};

struct Rows {
    const void* logits;
    uint64_t ld, rows, first;   // first: rows of earlier launches
    uint32_t vocab, parts, per; // per: vectors of a part
    uint32_t list;              // places that a part's list holds
    Part* part;                 // [rows, parts]
    uint64_t* lists;            // [rows, parts, list]: places, or masses up to each bin and counts of bins
    // settings: of all rows, or of each
    double temperature, top_p, min_p;
    int64_t top_k;
    const float *temperatures, *top_ps, *min_ps;
    const int64_t* top_ks;
    float* logps;
    int64_t* ids;
    const float* uniforms;
};

struct Settings {
    double t, top_p, min_p;
    uint32_t k;       // vocab: every word
    bool listed;      // by the parts' lists, else by masses
    bool filtered;    // of the latter: not every word is kept, and the parts leave histograms
};
// What the host knows of a call's rows: kListed and kFiltered as above, kWhole neither.
enum Kind { kEither, kListed, kFiltered, kWhole };
template <Kind kKind>
__device__ __forceinline__ Settings settings(const Rows& a, uint64_t row) {
    Settings s;
    s.t = a.temperatures != nullptr ? double(a.temperatures[row]) : a.temperature;
    s.top_p = a.top_ps != nullptr ? double(a.top_ps[row]) : a.top_p;
    s.min_p = a.min_ps != nullptr ? double(a.min_ps[row]) : a.min_p;
    const int64_t k = a.top_ks != nullptr ? a.top_ks[row] : a.top_k;
    s.k = k <= 0 || k >= int64_t(a.vocab) ? a.vocab : uint32_t(k);
    if (!(s.t > 0.0)) s.t = 1.0, s.k = 1;   // the largest
    s.t = fmin(fmax(s.t, 1e-30), 1e30);     // so that neither it nor its inverse is infinite in fp32
    s.listed = kKind == kListed || (kKind == kEither && s.k <= kMost);
    s.filtered = kKind == kFiltered || (kKind != kWhole && (s.top_p < 1.0 || s.k < a.vocab || s.min_p > 0.0));
    return s;
}

template <uint32_t kT, typename V, typename Op>
__device__ __forceinline__ V block_all(V v, V* shared, Op op) {   // the same value in every lane; shared: kT / 64
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v = op(v, __shfl_xor(v, d));
    if constexpr (kT == 64) return v;
    __syncthreads();   // whoever read it before has
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    v = shared[0];
#pragma unroll
    for (uint32_t w = 1; w < kT / 64; ++w) v = op(v, shared[w]);
    return v;
}
struct Max {
    __device__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct Add {
    template <typename V>
    __device__ V operator()(V a, V b) const { return a + b; }
};

__device__ __forceinline__ float bin_scale(double t) { return float(double(kBinsOfT) / t); }

// ---------------------------------------------------------------------
// What was read is used once more: no converted copies of it stay in registers meanwhile.
template <uint32_t kV>
__device__ __forceinline__ void afresh(u32x4 (&x)[kV]) {
#pragma unroll
    for (uint32_t i = 0; i < kV; ++i) asm volatile("" : "+v"(x[i]));
}

// Bound by its bytes: 4092 rows of 128256 bf16 245 us (4.3 TB/s; a device copy moves 4.95, a sum
// that only reads 3.7), 1023 x 50257 fp32 42 (4.9), 512 x 152064 fp32 72 (4.3).  Few rows wait for
// their own steps: 64 x 128256 18, one 7, 31 x 4096 5.6.  Parts are as large as registers allow, 8
// vectors of 256 lanes, since each leaves 1 to 6 KB that the row's join reads.
template <typename E, uint32_t kV, Kind kKind>
__global__ __launch_bounds__(kPartLanes) void rows_parts_kernel(const Rows a) {
    constexpr uint32_t kN = kOf<E>;
    __shared__ float shared_m[kPartLanes / 64];
    __shared__ double shared_s[kPartLanes / 64];
    __shared__ uint32_t count, hits;
    __shared__ float bound_of;
    __shared__ __attribute__((aligned(16))) uint64_t mass[kBins];
    __shared__ uint32_t number[kBins];
    static_assert(kPartLanes * 16 <= sizeof(mass) && kPartLanes <= kBins, "the vectors with candidates");
    float* const most = reinterpret_cast<float*>(mass);   // [kPartLanes]
    const uint64_t row = blockIdx.x / a.parts;
    const uint32_t part = blockIdx.x % a.parts;
    const Row<E> r(a.logits, a.ld, a.first + row, a.vocab);
    u32x4 x[kV];
    r.load(x, [&](uint32_t i) {
        const uint32_t in = i * kPartLanes + threadIdx.x;
        return in < a.per ? part * a.per + in : ~0u;
    });
    const Settings s = settings<kKind>(a, a.first + row);
    float mine = kNegInf, each[kV];   // the largest of each vector
#pragma unroll
    for (uint32_t i = 0; i < kV; ++i) {
        each[i] = item<E>(x[i], 0);
#pragma unroll
        for (uint32_t j = 1; j < kN; ++j) each[i] = fmaxf(each[i], item<E>(x[i], j));
        mine = fmaxf(mine, each[i]);
    }
    if (threadIdx.x == 0) count = 0, hits = 0;
    const float m = block_all<kPartLanes>(mine, shared_m, Max{});
    Part* const out = a.part + row * a.parts + part;
    uint64_t* const list = a.lists + (row * a.parts + part) * a.list;
    const float from = base(m);
    afresh(x);

    if (s.listed) {
        // 2^(c x - from c), from c rounded, which the sum makes up for at its end: below 2^24 that
        // is half an octave at most.  Of larger ones, a part of a finite mask's value or a low
        // temperature, 2^(c (x - from)): from 2^31 on the rounding alone leaves an exponential's range.
        const float c = float(double(kLog2e) / s.t);
        const bool far = !(fabsf(from * c) < 0x1p24f);
        const float less = far ? 0.0f : from * c;
        float sum = 0.0f;
        if (far) {
#pragma unroll
            for (uint32_t i = 0; i < kV; ++i)
#pragma unroll
                for (uint32_t j = 0; j < kN; ++j) sum += __builtin_amdgcn_exp2f((item<E>(x[i], j) - from) * c);
        } else {
#pragma unroll
            for (uint32_t i = 0; i < kV; ++i)
#pragma unroll
                for (uint32_t j = 0; j < kN; ++j) sum += __builtin_amdgcn_exp2f(fmaf(item<E>(x[i], j), c, -less));
        }
        afresh(x);
        // A bound with k words of the part or more above it: the k-th largest of the
        // lanes' maxima, to 16 bits.  Of 256 lanes about 256 ln(256 / (256 - k)) words are.
        most[threadIdx.x] = mine;
        const double total = block_all<kPartLanes>(double(sum), shared_s, Add{}) * (far ? 1.0 : exp2_wide(double(less) - double(from) * double(c)));
        if (threadIdx.x < 64) {
            uint32_t keys[kPartLanes / 64];
#pragma unroll
            for (uint32_t i = 0; i < kPartLanes / 64; ++i) keys[i] = key_of(most[i * 64 + threadIdx.x]) >> 16;
            uint32_t bound = 0;
#pragma unroll 1
            for (int bit = 15; bit >= 0; --bit) {
                const uint32_t with = bound | 1u << bit;
                uint32_t n = 0;
#pragma unroll
                for (uint32_t i = 0; i < kPartLanes / 64; ++i) n += __popcll(__ballot(keys[i] >= with));
                if (n >= s.k) bound = with;
                if (n == s.k) break;
            }
            if (threadIdx.x == 0) bound_of = float_of(bound << 16);
        }
        __syncthreads();   // also: the lanes' maxima have been read
        const float bound = bound_of;
        const auto keep = [&](float f, uint32_t at_v, uint32_t j) {
            if (f > kNegInf && !(f < bound)) {
                const uint32_t at = atomicAdd(&count, 1u);
                if (at < a.list) list[at] = place_of(f, r.index(at_v, j));
            }
        };
        // Few vectors have a candidate: those go to LDS, and then every lane looks at one word at a
        // time.  A bound of NaN's bits is that of fewer lanes than k: every word.
        u32x4* const found = reinterpret_cast<u32x4*>(mass);
        uint32_t* const found_v = number;
#pragma unroll
        for (uint32_t i = 0; i < kV; ++i)
            if (!(each[i] < bound) && each[i] > kNegInf) {
                const uint32_t at = atomicAdd(&hits, 1u);
                if (at < kPartLanes) found[at] = x[i], found_v[at] = part * a.per + i * kPartLanes + threadIdx.x;
            }
        __syncthreads();
        const uint32_t n = hits;
        if (n <= kPartLanes) {
            for (uint32_t i = threadIdx.x; i < n * kN; i += kPartLanes) {
                keep(item_at<E>(found[i / kN], i % kN), found_v[i / kN], i % kN);
            }
        } else {
#pragma unroll
            for (uint32_t i = 0; i < kV; ++i)
#pragma unroll
                for (uint32_t j = 0; j < kN; ++j) keep(item<E>(x[i], j), part * a.per + i * kPartLanes + threadIdx.x, j);
        }
        __syncthreads();
        if (threadIdx.x == 0) *out = Part{m, count, total};
        return;
    }
    const Weigh weigh(1.4426950408889634073599 / s.t, from);
    const float scale = bin_scale(s.t), top_bin = floorf(m * scale);
    if (s.filtered) {
        for (uint32_t i = threadIdx.x; i < kBins; i += kPartLanes) mass[i] = 0, number[i] = 0;
        __syncthreads();
    }
    // a part has at most 2^14 words: whole numbers of 2^-48
    double sum = 0.0;
    bool nan = false;
#pragma unroll
    for (uint32_t i = 0; i < kV; ++i) {
        asm volatile("" : "+v"(x[i]), "+v"(sum));   // a vector's words after the last one's: few registers
#pragma unroll
        for (uint32_t j = 0; j < kN; ++j) {
            const float f = item<E>(x[i], j);
            nan |= f != f;
            const double w = weigh(f);
            sum += w;
            if (s.filtered) {
                const float bin = top_bin - floorf(f * scale);
                if (bin >= 0.0f && bin < float(kBins)) {
                    atomicAdd(reinterpret_cast<unsigned long long*>(&mass[uint32_t(bin)]),
                              static_cast<unsigned long long>(w * 0x1p48 + 0.5));
                    atomicAdd(&number[uint32_t(bin)], 1u);
                }
            }
        }
    }
    if (nan) sum = __builtin_nan("");
    sum = block_all<kPartLanes>(sum, shared_s, Add{});
    if (s.filtered) {
        // the masses of all bins up to each
        static_assert(kBins == 2 * kPartLanes, "two bins a lane");
        const uint64_t one = mass[2 * threadIdx.x], two = one + mass[2 * threadIdx.x + 1];
        uint64_t upto = two;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint64_t below = __shfl_up(upto, d);
            if ((threadIdx.x & 63) >= uint32_t(d)) upto += below;
        }
        uint64_t* const waves = reinterpret_cast<uint64_t*>(shared_s);
        __syncthreads();
        if ((threadIdx.x & 63) == 63) waves[threadIdx.x >> 6] = upto;
        __syncthreads();
        for (uint32_t w = 0; w < threadIdx.x >> 6; ++w) upto += waves[w];
        list[2 * threadIdx.x] = upto - two + one, list[2 * threadIdx.x + 1] = upto;
        reinterpret_cast<uint32_t*>(list + kBins)[threadIdx.x] = number[2 * threadIdx.x] | number[2 * threadIdx.x + 1] << 16;
    }
    if (threadIdx.x == 0) *out = Part{m, 0, sum};
}

// ---------------------------------------------------------------------
// A row's parts joined.
struct Joined {
    float m;
    double sum;   // of exp((x - m) / T)
    bool bad;     // a NaN, an infinity, nothing but -inf
};
__device__ __forceinline__ double mass_of(const Part& p, float m, double c) {   // in that of the row's largest weight
    return p.m > kNegInf || p.sum != p.sum ? p.sum * exp2_wide((double(p.m) - double(m)) * c) : 0.0;
}
template <uint32_t kT>
__device__ __forceinline__ Joined join_parts(const Rows& a, const Part* part, double c, double* shared) {
    const Part own = threadIdx.x < a.parts ? part[threadIdx.x] : Part{kNegInf, 0, 0.0};
    float m = own.m;
    for (uint32_t p = threadIdx.x + kT; p < a.parts; p += kT) m = fmaxf(m, part[p].m);
    m = block_all<kT>(m, reinterpret_cast<float*>(shared), Max{});
    if (__builtin_isinf(m)) return {m, 0.0, true};
    double sum = mass_of(own, m, c);
    for (uint32_t p = threadIdx.x + kT; p < a.parts; p += kT) sum += mass_of(part[p], m, c);
    sum = block_all<kT>(sum, shared, Add{});
    return {m, sum, !(sum > 0.0)};
}

// What a row's workgroup has in LDS.
template <uint32_t kSorted_>
struct Shared {
    static constexpr uint32_t kSorted = kSorted_;   // candidates that it holds
    union {
        uint64_t places[kSorted];
        struct {
            uint64_t mass[1 << kDigit];
            uint32_t number[1 << kDigit];
        } digits;
    };
    uint64_t few[256];       // the k largest, sorted, or a border's neighbours
    double weights[kMost];
    double waves[16];        // of the block's sums
    uint64_t scan_m[16];
    uint32_t scan_n[16];
    uint32_t count, found_index, found_count, tied, held;
    uint64_t found;
    double found_mass;
};
// What a row that goes by histograms has beside it.
struct Bins {
    union {
        uint64_t mass[kBins];
        uint64_t sub_mass[kSubBins];
    };
    union {
        uint32_t number[kBins];
        uint32_t sub_number[kSubBins];
    };
    uint64_t kept[kMostParts];    // mass of each part
    double factor[kMostParts];    // 2^-44 of the row's largest weight in 2^-48 of the part's
    float offset[kMostParts];     // bins from the row's first to the part's
    float bin;                    // whose words are held; -1: none
};

// The bin, of kN in falling order, in which a running count or mass first comes to `reach`,
// `before` of it ahead of all bins; kN where none does.  Left in sh with what comes before it
// and its number of words.
template <uint32_t kT, uint32_t kN, typename Sh>
__device__ __forceinline__ void find_bin(const uint64_t* mass, const uint32_t* number, bool by_mass, uint64_t reach, uint64_t before_mass,
                         uint32_t before, Sh& sh) {
    constexpr uint32_t kEach = (kN + kT - 1) / kT;
    const uint32_t bin0 = threadIdx.x * kEach;
    uint64_t m = 0;
    uint32_t n = 0;
    for (uint32_t i = 0; i < kEach; ++i)
        if (bin0 + i < kN) m += mass[bin0 + i], n += number[bin0 + i];
    uint64_t upto_m = m;
    uint32_t upto_n = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t below_m = __shfl_up(upto_m, d);
        const uint32_t below_n = __shfl_up(upto_n, d);
        if ((threadIdx.x & 63) >= uint32_t(d)) upto_m += below_m, upto_n += below_n;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 63) sh.scan_m[threadIdx.x >> 6] = upto_m, sh.scan_n[threadIdx.x >> 6] = upto_n;
    if (threadIdx.x == 0) sh.found_index = kN;
    __syncthreads();
    uint64_t at_m = before_mass + upto_m - m;
    uint32_t at_n = upto_n - n;   // of these bins
#pragma unroll
    for (uint32_t w = 0; w < kT / 64; ++w)
        if (w < threadIdx.x >> 6) at_m += sh.scan_m[w], at_n += sh.scan_n[w];
    for (uint32_t i = 0; i < kEach && bin0 + i < kN; ++i) {
        const uint64_t next_m = at_m + mass[bin0 + i];
        const uint32_t next_n = at_n + number[bin0 + i];
        const uint64_t from = by_mass ? at_m : before + at_n, to = by_mass ? next_m : before + next_n;
        if (next_n > at_n && to >= reach && (from < reach || at_n == 0)) {
            sh.found_index = bin0 + i;
            sh.found = at_m, sh.found_count = before + at_n, sh.tied = next_n - at_n;
        }
        at_m = next_m, at_n = next_n;
    }
    __syncthreads();
}

// The words of a row in the order of their index: the weights of those that are `kept` are
// added up, and the first word that takes the sum above `target` is found; where rounding
// leaves none, the last with a weight.  Every wave has a run of the row's vectors from v0
// to v1.  share: the target is that of the whole sum.  kFew: a weight costs 20 operations in
// 64 bits, so a lane goes over its kept words alone; where every word is kept that is slower.
template <typename E, uint32_t kT, bool kFew, typename Weight, typename Kept, typename Sh>
__device__ __forceinline__ uint32_t find_word(const Row<E>& r, uint32_t v0, uint32_t v1, double target, bool share, Weight weigh,
                                              Kept kept, Sh& sh) {
    const auto each_kept = [&](const u32x4& x, uint32_t v, auto f) {   // f(weight, index), by rising index
        if constexpr (kFew) {
            uint32_t those = 0;
#pragma unroll
            for (uint32_t j = 0; j < kOf<E>; ++j) those |= uint32_t(kept(item<E>(x, j), r.index(v, j))) << j;
            for (; those != 0; those &= those - 1) {
                const uint32_t j = __ffs(those) - 1;
                f(weigh(item_at<E>(x, j)), r.index(v, j));
            }
        } else {
#pragma unroll
            for (uint32_t j = 0; j < kOf<E>; ++j) f(weigh(item<E>(x, j)), r.index(v, j));
        }
    };
    constexpr uint32_t kWaves = kT / 64, kAtOnce = 2;
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const uint32_t each = (v1 - v0 + kWaves - 1) / kWaves;
    const uint32_t from = min(v0 + wave * each, v1), to = min(from + each, v1);
    const bool once = each <= 64 * kAtOnce;   // a part's run: what is read and weighed first is kept
    double sum = 0.0, own[kAtOnce] = {};
    u32x4 x[kAtOnce];
    uint32_t last = 0;   // index + 1 of the last with a weight
    for (uint32_t v = from + lane; v < to; v += 64 * kAtOnce) {
        r.load(x, [&](uint32_t u) { return v + u * 64 < to ? v + u * 64 : ~0u; });
#pragma unroll
        for (uint32_t u = 0; u < kAtOnce; ++u) {
            own[u] = 0.0;
            each_kept(x[u], v + u * 64, [&](double w, uint32_t index) {
                if (w > 0.0) own[u] += w, last = index + 1;
            });
            sum += own[u];
        }
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        sum += __shfl_xor(sum, d);
        last = max(last, uint32_t(__shfl_xor(int(last), d)));
    }
    __syncthreads();
    if (lane == 0) sh.waves[wave] = sum;
    if (threadIdx.x == 0) sh.found_index = 0;
    __syncthreads();
    double before = 0.0, total = 0.0;
    for (uint32_t w = 0; w < kWaves; ++w) total += sh.waves[w];
    if (share) target *= total;
    uint32_t chosen = kWaves, fallback = 0;
    for (uint32_t w = 0; w < kWaves; ++w) {
        if (sh.waves[w] > 0.0) fallback = w;
        if (chosen == kWaves) {
            if (before + sh.waves[w] > target) chosen = w;
            else before += sh.waves[w];
        }
    }
    const bool whole = chosen == kWaves;   // rounding: the last word there is
    if (whole) chosen = fallback;
    if (wave == chosen) {
        uint32_t found = last;
        double rest = target - before;
        for (uint32_t v = from + lane, t = 0; !whole && v - lane < to; v += 64, ++t) {
            u32x4 one[1] = {t == 0 ? x[0] : x[1]};
            double mine = t == 0 ? own[0] : own[1];
            if (!once) {
                r.load(one, [&](uint32_t) { return v < to ? v : ~0u; });
                mine = 0.0;
                each_kept(one[0], v, [&](double w, uint32_t) { mine += w; });
            } else if (v >= to) {
                mine = 0.0;
            }
            double upto = mine;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const double below = __shfl_up(upto, d);
                if (lane >= uint32_t(d)) upto += below;
            }
            const uint64_t over = __ballot(upto > rest && mine > 0.0);
            if (over != 0) {   // its words, one a lane
                const int at = __ffsll(static_cast<unsigned long long>(over)) - 1;
                u32x4 those;
#pragma unroll
                for (uint32_t w = 0; w < 4; ++w) those[w] = __shfl(one[0][w], at);
                const uint32_t index = r.index(v - lane + at, lane);
                const float f = item_at<E>(those, lane % kOf<E>);
                const double w = lane < kOf<E> && kept(f, index) ? weigh(f) : 0.0;
                const double ahead = __shfl(upto, at) - __shfl(mine, at);
                double c = w;
#pragma unroll
                for (int d = 1; d < int(kOf<E>); d <<= 1) {
                    const double below = __shfl_up(c, d);
                    if (lane >= uint32_t(d)) c += below;
                }
                // the last of those whose forerunners do not exceed it, the first at least
                const uint64_t some = __ballot(w > 0.0), in = __ballot(w > 0.0 && ahead + (c - w) <= rest);
                const int pick = in != 0 ? 63 - __builtin_clzll(in) : __ffsll(static_cast<unsigned long long>(some)) - 1;
                if (int(lane) == pick) sh.found_index = index + 1;
                found = 0;
                break;
            }
            rest -= __shfl(upto, 63);
        }
        if (found != 0 && lane == 0) sh.found_index = found;
    }
    __syncthreads();
    const uint32_t index = sh.found_index;
    __syncthreads();
    return index - 1;
}

// For every word of the row.
template <typename E, uint32_t kT, typename F>
__device__ __forceinline__ void each_word(const Row<E>& r, F f) {
    constexpr uint32_t kAtOnce = 8;
    for (uint32_t v = threadIdx.x; v < r.vectors; v += kT * kAtOnce) {
        u32x4 x[kAtOnce];
        r.load(x, [&](uint32_t u) { return v + u * kT; });
#pragma unroll
        for (uint32_t u = 0; u < kAtOnce; ++u)
#pragma unroll
            for (uint32_t j = 0; j < kOf<E>; ++j) f(item<E>(x[u], j), r.index(v + u * kT, j));
    }
}

// The border of a row by passes over the digits of its words' keys: the place of the last
// word of the prefix that a count (so many words) or a mass (the words with less than `reach`
// before them) asks for, 0 for every word.  prefix_mass: of the prefix, or null.
template <typename E, uint32_t kT, typename Sh>
__device__ __forceinline__ uint64_t border_by_digits(const Row<E>& r, float m, double c, bool by_mass, double reach, double* prefix_mass,
                                     Sh& sh) {
    constexpr uint32_t kDigits = 1 << kDigit;
    // masses in whole numbers whose sum 62 bits hold
    const int bits = 62 - (32 - __builtin_clz(r.vocab));
    const double one = ldexp(1.0, bits);
    const Weigh weigh(c, m);
    const auto whole = [&](float f) { return uint64_t(weigh(f) * one + 0.5); };
    const uint64_t target = by_mass ? uint64_t(ceil(fmax(reach, 0.0) * one)) : uint64_t(reach);
    uint32_t prefix = 0, known = 0, before = 0;
    uint64_t before_mass = 0;
    while (known < 32) {
        const uint32_t left = 32 - known - kDigit;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < kDigits; i += kT) sh.digits.mass[i] = 0, sh.digits.number[i] = 0;
        __syncthreads();
        each_word<E, kT>(r, [&](float f, uint32_t) {
            if (!(f > kNegInf)) return;
            const uint32_t key = key_of(f);
            if (known > 0 && (key >> (32 - known)) != prefix) return;
            const uint32_t bin = kDigits - 1 - ((key >> left) & (kDigits - 1));   // falling
            atomicAdd(&sh.digits.number[bin], 1u);
            atomicAdd(reinterpret_cast<unsigned long long*>(&sh.digits.mass[bin]), static_cast<unsigned long long>(whole(f)));
        });
        __syncthreads();
        find_bin<kT, kDigits>(sh.digits.mass, sh.digits.number, by_mass, target, before_mass, before, sh);
        const uint32_t bin = sh.found_index;
        if (bin == kDigits) return 0;   // the row has less
        prefix = prefix << kDigit | (kDigits - 1 - bin);
        known += kDigit;
        before = sh.found_count, before_mass = sh.found;
    }
    const uint32_t tied = sh.tied;
    const uint64_t w = whole(float_of(prefix));
    uint64_t take = tied;
    if (!by_mass) take = target - before;
    else if (w > 0) take = target > before_mass ? (target - before_mass + w - 1) / w : 1;
    take = min(max(take, uint64_t(1)), uint64_t(tied));
    if (prefix_mass != nullptr) *prefix_mass = double(before_mass + w * take) / one;
    __syncthreads();
    if (take >= tied) return uint64_t(prefix) << 32;
    const uint32_t index = find_word<E, kT, true>(
        r, 0, r.vectors, double(take) - 0.5, false, [](float) { return 1.0; },
        [&](float f, uint32_t) { return f > kNegInf && key_of(f) == prefix; }, sh);
    return uint64_t(prefix) << 32 | uint32_t(~index);
}

// How many of the codes of 16-bit floats, in their order (code_of), lie below `t` times 1 / scale:
// those with scale x < t, rounded as the histograms have it.  Every wave by itself.
template <typename E>
__device__ __forceinline__ uint32_t codes_below(float t, float scale) {
    constexpr uint32_t kInf = (E::kNegInf & 0x7FFFu) | 0x8000u;   // +infinity's
    uint32_t below = 0;
#pragma unroll
    for (uint32_t step = 1024; step > 0; step = step == 1024 ? 16 : step == 16 ? 1 : 0) {
        const uint32_t lane = threadIdx.x & 63, u = below + lane * step + step - 1;
        const float x = E::lo(u & 0x8000u ? u & 0x7FFFu : ~u & 0xFFFFu);
        below += uint32_t(__popcll(__ballot(u < kInf && (step > 1 || lane < 16) && !(x * scale >= t)))) * step;
    }
    return below;
}
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef int16_t i16x2 __attribute__((ext_vector_type(2)));
// Of a pair of 16-bit floats a bit each, 0 and 16: whether its code is among `many` from `from` on.
__device__ __forceinline__ uint32_t codes_in(uint32_t pair, u16x2 from, u16x2 many) {
    const uint32_t sign = __builtin_bit_cast(uint32_t, __builtin_bit_cast(i16x2, pair) >> i16x2{15, 15});
    const u16x2 code = __builtin_bit_cast(u16x2, pair ^ (sign | 0x80008000u));   // all bits of a negative one turned
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_elementwise_sub_sat(many, u16x2(code - from)), u16x2{1, 1}));
}

// The words with lo <= scale x < lo + 1, into sh.places as many as it holds; how many there are.
// Found by bits, of 16-bit words two at a time by their codes, and put in place by one addition of
// a wave to the counter for 8 vectors of each lane: the index first, the logit read again.
template <typename E, uint32_t kT, typename Sh>
__device__ __forceinline__ uint32_t gather_bin(const Row<E>& r, float scale, float lo, Sh& sh) {
    constexpr bool kCodes = !std::is_same_v<E, F32>;
    constexpr uint32_t kAtOnce = 8, kMasks = kOf<E> / 4;   // of 32 bits: 8 vectors of 4, or 4 of 8
    __syncthreads();
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    u16x2 from, many;
    if constexpr (kCodes) {
        const uint32_t a = codes_below<E>(lo, scale), b = codes_below<E>(lo + 1.0f, scale);
        from = u16x2{uint16_t(a), uint16_t(a)}, many = u16x2{uint16_t(b - a), uint16_t(b - a)};
    }
    for (uint32_t v0 = 0; v0 < r.vectors; v0 += kT * kAtOnce) {
        const uint32_t v = v0 + threadIdx.x;
        u32x4 x[kAtOnce];
        r.load(x, [&](uint32_t u) { return v + u * kT; });
        uint32_t those[kMasks] = {}, n = 0;
#pragma unroll
        for (uint32_t u = 0; u < kAtOnce; ++u)
#pragma unroll
            for (uint32_t w = 0; w < 4; ++w) {
                if constexpr (kCodes) {
                    those[u / 4] |= codes_in(x[u][w], from, many) << (u % 4 * 4 + w);
                } else {
                    const float f = item<E>(x[u], w) * scale;
                    those[0] |= uint32_t(f >= lo && f < lo + 1.0f) << (u * 4 + w);
                }
            }
#pragma unroll
        for (uint32_t k = 0; k < kMasks; ++k) n += __popc(those[k]);
        uint32_t at = n;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t below = __shfl_up(at, d);
            if ((threadIdx.x & 63) >= uint32_t(d)) at += below;
        }
        const uint32_t all = __shfl(at, 63);
        if (all == 0) continue;
        uint32_t before = 0;
        if ((threadIdx.x & 63) == 0) before = atomicAdd(&sh.count, all);
        at += __shfl(before, 0) - n;
#pragma unroll
        for (uint32_t k = 0; k < kMasks; ++k)
            for (uint32_t m = those[k]; m != 0; m &= m - 1, ++at) {
                const uint32_t bit = __ffs(m) - 1, u = kCodes ? k * 4 + bit % 16 / 4 : bit / 4;
                const uint32_t j = kCodes ? bit % 4 * 2 + bit / 16 : bit % 4;
                if (at < Sh::kSorted) sh.places[at] = r.index(v + u * kT, j);
            }
    }
    __syncthreads();
    const uint32_t n = sh.count;
    for (uint32_t i = threadIdx.x; i < min(n, Sh::kSorted); i += kT) {
        const uint32_t index = uint32_t(sh.places[i]);
        sh.places[i] = place_of(r.at(index), index);
    }
    __syncthreads();
    return n;
}

// What the histograms of a row's parts say of it together.
__device__ __forceinline__ bool bins_do(const Rows& a, float top_bin) {
    // whole numbers of 2^-44 of a row of up to 2^18 words; bins that floats tell apart
    return a.vocab <= (1u << 18) && a.parts <= kMostParts && fabsf(top_bin) < 0x1p22f;
}
template <uint32_t kT>
__device__ __forceinline__ void join_bins(const Rows& a, const Part* part, const uint64_t* lists, float m, double c, float scale, float top_bin,
                          Bins& bins) {
    for (uint32_t i = threadIdx.x; i < kBins; i += kT) bins.mass[i] = 0, bins.number[i] = 0;
    if (threadIdx.x < a.parts) {
        const float mp = part[threadIdx.x].m;
        bins.factor[threadIdx.x] = mp > kNegInf ? exp2_wide((double(mp) - double(m)) * c) * 0x1p-4 : 0.0;
        bins.offset[threadIdx.x] = mp > kNegInf ? top_bin - floorf(mp * scale) : 2.0f * kBins;
    }
    __syncthreads();
    constexpr uint32_t kAtOnce = 4;
    for (uint32_t i0 = threadIdx.x; i0 < a.parts * kBins; i0 += kT * kAtOnce) {
        uint64_t upto[kAtOnce], below[kAtOnce];
        uint32_t number[kAtOnce];
#pragma unroll
        for (uint32_t u = 0; u < kAtOnce; ++u) {
            const uint32_t i = min(i0 + u * kT, a.parts * kBins - 1), p = i / kBins, bin = i % kBins;
            const uint64_t* const of = lists + uint64_t(p) * a.list;
            upto[u] = of[bin], below[u] = bin > 0 ? of[bin - 1] : 0;
            number[u] = reinterpret_cast<const uint16_t*>(of + kBins)[bin];
        }
#pragma unroll
        for (uint32_t u = 0; u < kAtOnce; ++u) {
            const uint32_t i = i0 + u * kT, p = min(i / kBins, a.parts - 1);
            const float at = bins.offset[p] + float(i % kBins);
            if (i >= a.parts * kBins || number[u] == 0 || !(at < float(kBins))) continue;
            atomicAdd(&bins.number[uint32_t(at)], number[u]);
            atomicAdd(reinterpret_cast<unsigned long long*>(&bins.mass[uint32_t(at)]),
                      static_cast<unsigned long long>(double(upto[u] - below[u]) * bins.factor[p] + 0.5));
        }
    }
    __syncthreads();
}

// The border, as border_by_digits gives it, from the parts' histograms: the bin it lies in,
// whose words are binned again, and of those a few sorted.  Leaves the bin's words in
// sh.places, sh.held of them, and its number in bins.bin.  false: what is looked for lies
// below the histograms, or the bin holds too many.
template <typename E, uint32_t kT, typename Sh>
__device__ __forceinline__ bool border_by_bins(const Rows& a, const Part* part, const uint64_t* lists, const Row<E>& r, float m, double t,
                               bool by_mass, double reach, uint64_t* border, double* prefix_mass, Sh& sh, Bins& bins) {
    const double c = 1.4426950408889634073599 / t;
    const float scale = bin_scale(t), top_bin = floorf(m * scale);
    __syncthreads();
    if (threadIdx.x == 0) bins.bin = -1.0f;
    if (!bins_do(a, top_bin)) return false;
    const uint64_t target = by_mass ? uint64_t(ceil(fmax(reach, 0.0) * 0x1p44)) : uint64_t(reach);
    join_bins<kT>(a, part, lists, m, c, scale, top_bin, bins);
    find_bin<kT, kBins>(bins.mass, bins.number, by_mass, target, 0, 0, sh);
    const uint32_t bin = sh.found_index, n = sh.tied, before = sh.found_count;
    const uint64_t before_mass = sh.found;
    if (bin == kBins || n > Sh::kSorted) return false;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < kSubBins; i += kT) bins.sub_mass[i] = 0, bins.sub_number[i] = 0;
    const float lo = top_bin - float(bin);   // floor(v) == lo
    if (gather_bin<E, kT>(r, scale, lo, sh) != n) return false;
    if (threadIdx.x == 0) sh.held = n, bins.bin = float(bin);
    const auto sub_of = [&](float f) { return kSubBins - 1 - min(uint32_t((f * scale - lo) * float(kSubBins)), kSubBins - 1); };
    const Weigh weight(c, m);
    for (uint32_t i = threadIdx.x; i < n; i += kT) {
        const float f = logit_of(sh.places[i]);
        atomicAdd(&bins.sub_number[sub_of(f)], 1u);
        atomicAdd(reinterpret_cast<unsigned long long*>(&bins.sub_mass[sub_of(f)]),
                  static_cast<unsigned long long>(weight(f) * 0x1p44 + 0.5));
    }
    __syncthreads();
    find_bin<kT, kSubBins>(bins.sub_mass, bins.sub_number, by_mass, target, before_mass, before, sh);
    const uint32_t sub = sh.found_index, few = sh.tied, before_sub = sh.found_count;
    const double mass_sub = double(sh.found) * 0x1p-44;
    if (sub == kSubBins) return false;   // a rounding at the end of the bin
    __syncthreads();
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += kT)
        if (sub_of(logit_of(sh.places[i])) == sub) {
            const uint32_t at = atomicAdd(&sh.count, 1u);
            if (at < 64) sh.few[at] = sh.places[i];
        }
    __syncthreads();
    if (few > 64) {
        // Equal words, as 16-bit logits have them by the hundreds: as many as are asked for, by
        // their index, whose bits are binned in turn.
        const uint32_t key = uint32_t(sh.few[0] >> 32);
        const double w = weight(float_of(key));
        double more = by_mass ? ceil((reach - mass_sub) / w) : reach - double(before_sub);
        const uint32_t take = more < 1.0 ? 1 : more < double(few) ? uint32_t(more) : few;
        const uint32_t shift = max(0, 32 - 10 - __builtin_clz(max(r.vocab - 1, 1u)));   // of an index, to 1024 bins
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < kSubBins; i += kT) bins.sub_mass[i] = 0, bins.sub_number[i] = 0;
        if (threadIdx.x == 0) sh.count = 0;
        __syncthreads();
        bool other = false;
        for (uint32_t i = threadIdx.x; i < n; i += kT) {
            const uint64_t place = sh.places[i];
            if (uint32_t(place >> 32) == key) atomicAdd(&bins.sub_number[index_of(place) >> shift], 1u);
            else other |= sub_of(logit_of(place)) == sub;
        }
        if (__syncthreads_or(other)) return false;
        find_bin<kT, kSubBins>(bins.sub_mass, bins.sub_number, false, take, 0, 0, sh);
        const uint32_t among = sh.found_index, ahead = sh.found_count;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < n; i += kT)
            if (uint32_t(sh.places[i] >> 32) == key && index_of(sh.places[i]) >> shift == among)
                sh.few[atomicAdd(&sh.count, 1u)] = sh.places[i];   // at most 2^8 indices
        __syncthreads();
        if (threadIdx.x < sh.count) {
            const uint64_t own = sh.few[threadIdx.x];
            uint32_t rank = 0;
            const uint32_t all = sh.count;
#pragma unroll 8
            for (uint32_t i = 0; i < all; ++i) rank += sh.few[i] > own;
            if (ahead + rank + 1 == take) sh.found = own;
        }
        if (threadIdx.x == 0) sh.found_mass = mass_sub + w * take;
    } else if (threadIdx.x < 64) {
        const uint32_t lane = threadIdx.x;
        const uint64_t own = lane < few ? sh.few[lane] : 0;
        uint32_t rank = 0;
#pragma unroll 8
        for (uint32_t i = 0; i < few; ++i) rank += sh.few[i] > own;
        if (lane < few) sh.few[64 + rank] = own;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const uint64_t place = lane < few ? sh.few[64 + lane] : 0;
        const double w = lane < few ? weight(logit_of(place)) : 0.0;
        double upto = w;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const double below = __shfl_up(upto, d);
            if (lane >= uint32_t(d)) upto += below;
        }
        // the first of them at least: their bin was reached
        const bool in = lane < few && (lane == 0 || (by_mass ? mass_sub + (upto - w) < reach : double(before_sub + lane) < reach));
        const int end = 63 - __builtin_clzll(__ballot(in));
        const uint64_t last = __shfl(place, end);
        const double mass = mass_sub + __shfl(upto, end);
        if (lane == 0) sh.found = last, sh.found_mass = mass;
    }
    __syncthreads();
    *border = sh.found;
    if (prefix_mass != nullptr) *prefix_mass = sh.found_mass;
    __syncthreads();
    return true;
}

// ---------------------------------------------------------------------
// The k largest words of a row, sorted in sh.few; how many there are (-inf are none).
//
// One wave picks them from the parts' lists, up to 16 words a lane at a time: a key that k and
// at most 128 of them reach, bit by bit, by counting ballots, and where more are equal the bits of
// their index (by passes over the row such a row took 110 us); those go on to the next lists and
// are ranked by counting in the end.  Others than the first wave wait.
// ---------------------------------------------------------------------
constexpr uint32_t kPicked = 1024;
template <typename Sh>
__device__ __forceinline__ bool pick_largest(const Rows& a, const Part* part, const uint64_t* lists, uint32_t k, Sh& sh) {
    static_assert(Sh::kSorted >= kPicked, "it holds them");
    constexpr uint32_t kEach = kPicked / 64;
    const uint32_t lane = threadIdx.x;
    uint32_t n = 0, p = 0;
    do {
        // the next lists, as many of up to 64 as fit, a word a lane in turn; all on their way at once
        const uint32_t in = p + lane < a.parts ? part[p + lane].count : 0;
        if (__ballot(in > a.list) != 0) return false;
        uint32_t end = in;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t below = __shfl_up(end, d);
            if (lane >= uint32_t(d)) end += below;
        }
        const uint32_t took = min(uint32_t(__popcll(__ballot(n + end <= kPicked))), a.parts - p);   // ends only rise
        const uint32_t more = took > 0 ? __shfl(end, took - 1) : 0;
        uint64_t next[kEach];
        uint32_t of[kEach], from[kEach];
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) of[i] = from[i] = 0;
        for (uint32_t q = 0; q + 1 < took; ++q) {
            const uint32_t edge = __builtin_amdgcn_readlane(end, q);
#pragma unroll
            for (uint32_t i = 0; i < kEach; ++i)
                if (i * 64 + lane >= edge) of[i] = q + 1, from[i] = edge;
        }
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            const uint32_t at = i * 64 + lane;
            next[i] = at < more ? lists[uint64_t(p + of[i]) * a.list + at - from[i]] : 0;
        }
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i)
            if (i * 64 + lane < more) sh.places[n + i * 64 + lane] = next[i];
        p += took, n += more;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (n <= k && p < a.parts) return false;   // a list does not fit beside so few
        if (n <= k) break;
        uint32_t keys[kEach];
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) keys[i] = i * 64 + lane < n ? uint32_t(sh.places[i * 64 + lane] >> 32) : 0;
        // from the first bit on in which they differ
        uint32_t low = ~0u, high = 0;
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) high = max(high, keys[i]), low = min(low, i * 64 + lane < n ? keys[i] : ~0u);
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) {
            high = max(high, uint32_t(__shfl_xor(int(high), d)));
            low = min(low, uint32_t(__shfl_xor(int(low), d)));
        }
        const int differ = high == low ? -1 : 31 - __builtin_clz(high ^ low);
        uint32_t bound = differ < 0 ? low : differ == 31 ? 0 : low >> (differ + 1) << (differ + 1), reached = n;
#pragma unroll 1
        for (int bit = differ; bit >= 0 && reached > kMost; --bit) {
            const uint32_t with = bound | 1u << bit;
            uint32_t have = 0;
#pragma unroll
            for (uint32_t i = 0; i < kEach; ++i) have += __popcll(__ballot(keys[i] >= with));
            if (have >= k) bound = with, reached = have;
        }
        uint32_t bound_low = 0;
        if (reached > kMost) {   // equal words, the first of them by the bits of their index
            bound_low = ~0u << (32 - __builtin_clz(max(a.vocab - 1, 1u)));
#pragma unroll 1
            for (uint32_t bit = ~bound_low / 2 + 1; reached > kMost; bit /= 2) {
                const uint64_t with = uint64_t(bound) << 32 | bound_low | bit;
                uint32_t have = 0;
#pragma unroll
                for (uint32_t i = 0; i < kEach; ++i) have += __popcll(__ballot(i * 64 + lane < n && sh.places[i * 64 + lane] >= with));
                if (have >= k) bound_low |= bit, reached = have;
            }
        }
        // in any order, each before where it was
        uint32_t at = 0;
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            const uint64_t own = i * 64 + lane < n ? sh.places[i * 64 + lane] : 0;
            const bool in = i * 64 + lane < n && own >= (uint64_t(bound) << 32 | bound_low);
            const uint64_t place = in ? own : 0, those = __ballot(in);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            if (in) sh.places[at + __popcll(those & ((uint64_t(1) << lane) - 1))] = place;
            at += __popcll(those);
        }
        n = reached;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    } while (p < a.parts);
    static_assert(kMost == 128, "two words a lane");
    const uint64_t own0 = lane < n ? sh.places[lane] : 0, own1 = lane + 64 < n ? sh.places[lane + 64] : 0;
    uint32_t rank0 = 0, rank1 = 0;
#pragma unroll 8
    for (uint32_t i = 0; i < n; ++i) {
        const uint64_t other = sh.places[i];
        rank0 += other > own0, rank1 += other > own1;
    }
    if (lane < n && rank0 < k) sh.few[rank0] = own0;
    if (lane + 64 < n && rank1 < k) sh.few[rank1] = own1;
    if (lane == 0) sh.held = min(n, k);
    return true;
}
template <typename E, uint32_t kT, typename Sh>
__device__ __forceinline__ uint32_t largest(const Rows& a, const Part* part, const uint64_t* lists, const Row<E>& r, float m, double c, uint32_t k,
                            Sh& sh) {
    __syncthreads();
    if (threadIdx.x < 64) {
        const bool done = pick_largest(a, part, lists, k, sh);
        if (threadIdx.x == 0 && !done) sh.held = ~0u;
    }
    __syncthreads();
    if (sh.held != ~0u) return sh.held;
    const uint64_t border = border_by_digits<E, kT>(r, m, c, false, double(k), nullptr, sh);
    __syncthreads();
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    each_word<E, kT>(r, [&](float f, uint32_t index) {
        if (f > kNegInf && place_of(f, index) >= border) {
            const uint32_t at = atomicAdd(&sh.count, 1u);
            if (at < kMost) sh.few[128 + at] = place_of(f, index);
        }
    });
    __syncthreads();
    const uint32_t n = min(sh.count, k);
    for (uint32_t i = threadIdx.x; i < n; i += kT) {
        const uint64_t own = sh.few[128 + i];
        uint32_t rank = 0;
        for (uint32_t j = 0; j < n; ++j) rank += sh.few[128 + j] > own;
        sh.few[rank] = own;
    }
    __syncthreads();
    return n;
}

// Bound by the wave's steps, one after the other: 31 rows of one part 6.5 us, 1023 of 7 parts and k
// = 128 23, 4092 of 8 and k = 64 29.  One wave, since 1024 lanes met at a barrier after each step.
constexpr uint32_t kListedLanes = 64;
template <typename E>
__global__ __launch_bounds__(kListedLanes) void top_rows_kernel(const Rows a) {
    __shared__ Shared<kPicked> sh;
    const uint64_t row = blockIdx.x, of = a.first + row;
    const Part* const part = a.part + row * a.parts;
    const uint64_t* const lists = a.lists + row * a.parts * a.list;
    const Settings s = settings<kListed>(a, of);
    const uint32_t k = uint32_t(a.top_k);
    const double c = 1.4426950408889634073599 / s.t;
    const Joined j = join_parts<kListedLanes>(a, part, c, sh.waves);
    float* const logps = a.logps + of * k;
    int64_t* const ids = a.ids + of * k;
    if (j.bad) {
        for (uint32_t i = threadIdx.x; i < k; i += kListedLanes) logps[i] = __builtin_nanf(""), ids[i] = -1;
        return;
    }
    const Row<E> r(a.logits, a.ld, of, a.vocab);
    const uint32_t n = largest<E, kListedLanes>(a, part, lists, r, j.m, c, k, sh);
    const double lse = log(j.sum);
    for (uint32_t i = threadIdx.x; i < n; i += kListedLanes) {
        logps[i] = float((double(logit_of(sh.few[i])) - double(j.m)) / s.t - lse);
        ids[i] = index_of(sh.few[i]);
    }
    // words of probability 0 in the order of their index
    for (uint32_t done = n, v0 = 0; done < k && v0 < a.vocab; v0 += 64) {
        const uint32_t index = v0 + threadIdx.x;
        bool none = false;
        if (index < a.vocab) {
            if constexpr (std::is_same_v<E, F32>) none = r.x[index] == 0xFF800000u;
            else none = r.x[index] == E::kNegInf;
        }
        const uint64_t those = __ballot(none);
        const uint32_t at = done + __popcll(those & ((uint64_t(1) << threadIdx.x) - 1));
        if (none && at < k) logps[at] = kNegInf, ids[at] = index;
        done += __popcll(those);
    }
}

// ---------------------------------------------------------------------
// A draw from the k largest words, by the first wave: two words a lane, in their order.
template <typename E, uint32_t kT, typename Sh>
__device__ __forceinline__ void draw_listed(const Rows& a, uint64_t of, const Settings& s, const Part* part, const uint64_t* lists,
                            const Joined& j, double c, double u, double least, double lse, Sh& sh) {
    const Row<E> r(a.logits, a.ld, of, a.vocab);
    const uint32_t n = largest<E, kT>(a, part, lists, r, j.m, c, s.k, sh);
    if (threadIdx.x >= 64) return;
    const uint32_t lane = threadIdx.x;
    uint64_t place[2];
    double d[2], w[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const uint32_t i = 2 * lane + e;
        place[e] = i < n ? sh.few[i] : 0;
        d[e] = i < n ? double(logit_of(place[e])) - double(j.m) : 0.0;
        w[e] = i < n ? exp2_wide(d[e] * c) : 0.0;
    }
    double upto = w[0] + w[1];
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const double below = __shfl_up(upto, d);
        if (lane >= uint32_t(d)) upto += below;
    }
    const double total = __shfl(upto, 63);
    const double before[2] = {upto - w[1] - w[0], upto - w[1]};
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const uint32_t i = 2 * lane + e;
        const bool kept = i < n && (i == 0 || !(s.top_p < 1.0) || before[e] < s.top_p * total) && d[e] >= least;
        w[e] = kept ? w[e] : 0.0;
        sh.weights[i] = w[e];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const uint32_t index[2] = {index_of(place[0]), index_of(place[1])};
    double mass = 0.0, sums[2] = {0.0, 0.0};   // in one order everywhere
#pragma unroll 8
    for (uint32_t i = 0; i < n; ++i) {
        const double v = sh.weights[i];
        const uint32_t at = index_of(sh.few[i]);
        mass += v;
        if (at <= index[0]) sums[0] += v;
        if (at <= index[1]) sums[1] += v;
    }
    // the first word above the target, by its index; where rounding leaves none, the last
    uint32_t first = ~0u, last = 0;
#pragma unroll
    for (int e = 0; e < 2; ++e)
        if (w[e] > 0.0) {
            if (sums[e] > u * mass) first = min(first, index[e]);
            last = max(last, index[e]);
        }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        first = min(first, uint32_t(__shfl_xor(int(first), d)));
        last = max(last, uint32_t(__shfl_xor(int(last), d)));
    }
    const uint32_t chosen = first != ~0u ? first : last;
#pragma unroll
    for (int e = 0; e < 2; ++e)
        if (w[e] > 0.0 && index[e] == chosen) a.ids[of] = chosen, a.logps[of] = float(d[e] / s.t - lse);
}

// What a draw is by: its share of the mass, below 1 (what is no number is 0), and the least x -
// max that min_p allows.
__device__ __forceinline__ double share_of(float u) { return u > 0.0f ? double(fminf(u, 0x1.fffffep-1f)) : 0.0; }
__device__ __forceinline__ double least_of(const Settings& s) {
    return s.min_p > 0.0 ? fmin(log(s.min_p), 0.0) * s.t : -__builtin_inf();
}

// As top_rows_kernel; a row of 8 parts 11 us.
template <typename E>
__global__ __launch_bounds__(kListedLanes) void draw_listed_kernel(const Rows a) {
    __shared__ Shared<kPicked> sh;
    const uint64_t row = blockIdx.x, of = a.first + row;
    const Part* const part = a.part + row * a.parts;
    const uint64_t* const lists = a.lists + row * a.parts * a.list;
    const Settings s = settings<kListed>(a, of);
    const double c = 1.4426950408889634073599 / s.t;
    const Joined j = join_parts<kListedLanes>(a, part, c, sh.waves);
    if (j.bad) {
        if (threadIdx.x == 0) a.ids[of] = -1, a.logps[of] = __builtin_nanf("");
        return;
    }
    draw_listed<E, kListedLanes>(a, of, s, part, lists, j, c, share_of(a.uniforms[of]), least_of(s), log(j.sum), sh);
}

// The mass that each part keeps with a border in bin `at`: its bins above, and of that bin's words
// those up to the border.
template <typename E, uint32_t kT, typename Sh>
__device__ __forceinline__ void kept_by_parts(const Rows& a, const uint64_t* lists, const Row<E>& r, float m, double c, float scale, float top_bin,
                              float at, uint64_t border, Sh& sh, Bins& bins) {
    __syncthreads();
    if (threadIdx.x < a.parts) {
        const float above = at - bins.offset[threadIdx.x];   // bins of the part
        bins.kept[threadIdx.x] = !(above >= 1.0f) ? 0 : uint64_t(
            double(lists[uint64_t(threadIdx.x) * a.list + uint32_t(above) - 1]) * bins.factor[threadIdx.x] + 0.5);
    }
    __syncthreads();
    const Weigh weigh(c, m);
    const auto add = [&](uint64_t place) {
        const uint64_t mass = uint64_t(weigh(logit_of(place)) * 0x1p44 + 0.5);
        const uint32_t p = (index_of(place) + r.shift) / kOf<E> / a.per;
        atomicAdd(reinterpret_cast<unsigned long long*>(&bins.kept[p]), static_cast<unsigned long long>(mass));
    };
    uint32_t n = sh.held;
    if (bins.bin != at) n = gather_bin<E, kT>(r, scale, top_bin - at, sh);
    if (n <= Sh::kSorted) {
        for (uint32_t i = threadIdx.x; i < n; i += kT)
            if (sh.places[i] >= border) add(sh.places[i]);
    } else {
        const float lo = top_bin - at;
        each_word<E, kT>(r, [&](float f, uint32_t index) {
            const float v = f * scale;
            if (v >= lo && v < lo + 1.0f && place_of(f, index) >= border) add(place_of(f, index));
        });
    }
    __syncthreads();
}

template <typename E>
__device__ __forceinline__ void write_draw(const Rows& a, uint64_t of, const Row<E>& r, uint32_t index, const Joined& j, const Settings& s) {
    a.ids[of] = index;
    a.logps[of] = float((double(r.at(index)) - double(j.m)) / s.t - log(j.sum));
}

// The part in which the running mass exceeds u times all (sum_up: their sum, of up to 64 parts), and
// what of that mass lies within it; where rounding leaves none, the last with a mass and infinity.
template <typename Mass, typename Sh>
__device__ __forceinline__ double choose_part(const Rows& a, double u, bool sum_up, double all, Mass mass, uint32_t* chosen, Sh& sh) {
    if (threadIdx.x < 64) {
        const uint32_t lane = threadIdx.x;
        double before = 0.0, rest = __builtin_inf();
        uint32_t last = 0;
        for (uint32_t p = 0; p < a.parts; p += 64) {
            const double own = p + lane < a.parts ? mass(p + lane) : 0.0;
            double upto = own;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const double below = __shfl_up(upto, d);
                if (lane >= uint32_t(d)) upto += below;
            }
            const double total = __shfl(upto, 63);
            if (sum_up) all = total;
            const uint64_t some = __ballot(own > 0.0), over = __ballot(own > 0.0 && before + upto > u * all);
            if (over != 0) {
                const int at = __ffsll(static_cast<unsigned long long>(over)) - 1;
                last = p + at;
                rest = u * all - (before + __shfl(upto, at) - __shfl(own, at));
                break;
            }
            if (some != 0) last = p + 63 - __builtin_clzll(some);
            before += total;
        }
        if (lane == 0) sh.found_index = last, sh.found_mass = rest;
    }
    __syncthreads();
    *chosen = sh.found_index;
    const double rest = sh.found_mass;
    __syncthreads();
    return rest;
}

// A draw from all of a row's words: the parts' masses say which part it is in, which is read
// again.  Bound by latency: 512 x 152064 fp32 15 us.
constexpr uint32_t kWholeLanes = 256;
template <typename E>
__global__ __launch_bounds__(kWholeLanes) void draw_whole_kernel(const Rows a) {
    __shared__ Shared<1> sh;
    const uint64_t row = blockIdx.x, of = a.first + row;
    const Part* const part = a.part + row * a.parts;
    const Settings s = settings<kWhole>(a, of);
    const double c = 1.4426950408889634073599 / s.t;
    const Joined j = join_parts<kWholeLanes>(a, part, c, sh.waves);
    if (j.bad) {
        if (threadIdx.x == 0) a.ids[of] = -1, a.logps[of] = __builtin_nanf("");
        return;
    }
    const Row<E> r(a.logits, a.ld, of, a.vocab);
    uint32_t v0;
    const double target = choose_part(a, share_of(a.uniforms[of]), false, j.sum, [&](uint32_t p) { return mass_of(part[p], j.m, c); }, &v0, sh);
    v0 = min(v0 * a.per, r.vectors);
    const Weigh weigh(c, j.m);
    const uint32_t index = min(find_word<E, kWholeLanes, false>(
        r, v0, min(v0 + a.per, r.vectors), target, false, weigh, [](float, uint32_t) { return true; }, sh), a.vocab - 1);
    if (threadIdx.x == 0) write_draw(a, of, r, index, j, s);
}

// A draw by masses, or by each row's own settings.  Bound by latency, a workgroup a row: 64 rows of
// 128256 bf16, top_p 0.95, 40 us, of which the histograms joined and searched 7, the border bin's
// words 9 to 11 (the row read again), those binned and sorted 5 to 9, the word found in its part 6 to
// 10; 255 rows of 50257 fp16 with settings of their own 43.
template <typename E, Kind kKind, uint32_t kDrawLanes>
__global__ __launch_bounds__(kDrawLanes) void draw_rows_kernel(const Rows a) {
    __shared__ Shared<7680> sh;
    __shared__ Bins bins;
    const uint64_t row = blockIdx.x, of = a.first + row;
    const Part* const part = a.part + row * a.parts;
    const uint64_t* const lists = a.lists + row * a.parts * a.list;
    const Settings s = settings<kKind>(a, of);
    const double c = 1.4426950408889634073599 / s.t;
    const Joined j = join_parts<kDrawLanes>(a, part, c, sh.waves);
    if (j.bad) {
        if (threadIdx.x == 0) a.ids[of] = -1, a.logps[of] = __builtin_nanf("");
        return;
    }
    const double u = share_of(a.uniforms[of]), least = least_of(s);
    if (kKind == kEither && s.listed)
        return draw_listed<E, kDrawLanes>(a, of, s, part, lists, j, c, u, least, log(j.sum), sh);
    const Row<E> r(a.logits, a.ld, of, a.vocab);
    const Weigh weight(c, j.m);
    uint64_t border = 0;
    bool by_parts = true;   // their masses say which one it is in
    if (s.filtered) {
        double mass = j.sum;
        if (s.k < a.vocab) {
            if (!border_by_bins<E, kDrawLanes>(a, part, lists, r, j.m, s.t, false, double(s.k), &border, &mass, sh, bins)) {
                border = border_by_digits<E, kDrawLanes>(r, j.m, c, false, double(s.k), &mass, sh);
                if (threadIdx.x == 0) bins.bin = -1.0f;   // its words are no longer there
            }
            if (border == 0) mass = j.sum;
        }
        if (s.top_p < 1.0) {
            const double reach = s.top_p * mass;
            uint64_t nucleus = 0;
            if (!border_by_bins<E, kDrawLanes>(a, part, lists, r, j.m, s.t, true, reach, &nucleus, nullptr, sh, bins)) {
                nucleus = border_by_digits<E, kDrawLanes>(r, j.m, c, true, reach, nullptr, sh);
                if (threadIdx.x == 0) bins.bin = -1.0f;
            }
            border = max(border, nucleus);
        } else if (s.k == a.vocab) {
            if (threadIdx.x == 0) bins.bin = -1.0f;
        }
        if (s.min_p > 0.0) {   // the least logit that it allows
            const double x = double(j.m) + least;
            float f = float(x);
            if (double(f) - double(j.m) < least) f = float_of(key_of(f) + 1);
            border = max(border, uint64_t(key_of(f)) << 32);
        }
        const float scale = bin_scale(s.t), top_bin = floorf(j.m * scale);
        const float at = border != 0 ? top_bin - floorf(logit_of(border) * scale) : float(kBins);
        by_parts = bins_do(a, top_bin) && at < float(kBins);
        if (by_parts) {
            if (s.k == a.vocab && !(s.top_p < 1.0)) join_bins<kDrawLanes>(a, part, lists, j.m, c, scale, top_bin, bins);
            kept_by_parts<E, kDrawLanes>(a, lists, r, j.m, c, scale, top_bin, at, border, sh, bins);
        }
    }
    uint32_t v0 = 0, v1 = r.vectors;
    double target = u;
    if (by_parts) {
        if (s.filtered)
            target = choose_part(a, u, true, 0.0, [&](uint32_t p) { return double(bins.kept[p]) * 0x1p-44; }, &v0, sh);
        else
            target = choose_part(a, u, false, j.sum, [&](uint32_t p) { return mass_of(part[p], j.m, c); }, &v0, sh);
        v0 = min(v0 * a.per, r.vectors), v1 = min(v0 + a.per, r.vectors);
    }
    const float from = border != 0 ? logit_of(border) : kNegInf;
    const uint32_t index = find_word<E, kDrawLanes, true>(
        r, v0, v1, target, !by_parts, weight,
        [&](float f, uint32_t i) { return f > kNegInf && f >= from && place_of(f, i) >= border; }, sh);
    if (threadIdx.x == 0) write_draw(a, of, r, min(index, a.vocab - 1), j, s);
}

// ---------------------------------------------------------------------
struct Plan {
    uint32_t parts, per, list, lane;   // lane: vectors of a lane
};
Plan plan_of(size_t vocab, int dtype) {
    const uint64_t of = dtype == SF_DTYPE_F32 ? 4 : 8, vectors = (vocab + 2 * of - 2) / of;
    const uint64_t most = kPartLanes * kPartVectors, parts = (vectors + most - 1) / most, per = (vectors + parts - 1) / parts;
    uint32_t lane = 1;
    while (lane * kPartLanes < per) lane *= 2;
    return {uint32_t(parts), uint32_t(per), parts == 1 ? 2 * kList : kList, lane};
}
// Rows of more than 8192 vectors, not more of them than compute units, are drawn from by 1024 lanes:
// few waits to read a row. Otherwise 512, of which a compute unit has two rows and whose registers
// hold all.  A call in us, 512 | 1024: 64 x 128256 bf16 62.8 | 58.2, 1 x 139482 fp32 52.5 | 50.4;
// 377 x 121933 bf16 139 | 157, 351 x 2572 fp32 41 | 58, 221 x 1313 bf16 28 | 32.
constexpr uint32_t kWideRows = 256, kWideParts = 5;
// Rows of one pair of launches: 256 MiB of lists.
uint64_t rows_at_once(const Plan& p) {
    const uint64_t rows = (uint64_t(256) << 20) / (uint64_t(p.parts) * (8 * p.list + sizeof(Part)));
    return rows > 0 ? rows : 1;
}

template <typename E, Kind kKind>
int launch_rows(const Rows& a, uint32_t rows, uint32_t lane, bool top, hipStream_t st) {
    const auto kernel = lane == 1   ? rows_parts_kernel<E, 1, kKind>
                        : lane == 2 ? rows_parts_kernel<E, 2, kKind>
                        : lane == 4 ? rows_parts_kernel<E, 4, kKind>
                                    : rows_parts_kernel<E, 8, kKind>;
    hipLaunchKernelGGL(kernel, dim3(rows * a.parts), dim3(kPartLanes), 0, st, a);
    const int e = status();
    if (e != SF_OK) return e;
    if constexpr (kKind == kListed) {
        const auto join = top ? top_rows_kernel<E> : draw_listed_kernel<E>;
        hipLaunchKernelGGL(join, dim3(rows), dim3(kListedLanes), 0, st, a);
    } else if constexpr (kKind == kWhole) {
        hipLaunchKernelGGL(draw_whole_kernel<E>, dim3(rows), dim3(kWholeLanes), 0, st, a);
    } else {
        const bool wide = rows <= kWideRows && a.parts >= kWideParts;
        hipLaunchKernelGGL((wide ? draw_rows_kernel<E, kKind, 1024> : draw_rows_kernel<E, kKind, 512>), dim3(rows),
                           dim3(wide ? 1024 : 512), 0, st, a);
    }
    return status();
}

template <typename E>
int run_rows(Rows a, const Plan& p, bool top, hipStream_t st) {
    // a row's own temperature may ask for its largest word, its own top_k for a list
    const bool either = a.temperatures != nullptr || a.top_ks != nullptr;
    const bool filtered = a.top_ps != nullptr || a.min_ps != nullptr || a.top_p < 1.0 || a.min_p > 0.0 ||
                          (a.top_k > 0 && a.top_k < int64_t(a.vocab));
    const bool listed = !(a.temperature > 0.0) || (a.top_k > 0 && a.top_k <= int64_t(kMost)) || a.vocab <= kMost;
    const uint64_t most = rows_at_once(p);
    for (uint64_t r = 0; r < a.rows; r += most) {
        const uint32_t n = uint32_t(a.rows - r < most ? a.rows - r : most);
        a.first = r;
        const int e = either     ? launch_rows<E, kEither>(a, n, p.lane, top, st)
                      : listed   ? launch_rows<E, kListed>(a, n, p.lane, top, st)
                      : filtered ? launch_rows<E, kFiltered>(a, n, p.lane, top, st)
                                 : launch_rows<E, kWhole>(a, n, p.lane, top, st);
        if (e != SF_OK) return e;
    }
    return SF_OK;
}

int check_rows(const Rows& a, int dtype, const void* work) {
    if (a.logits == nullptr || a.logps == nullptr || a.ids == nullptr || work == nullptr) return SF_EINVAL;
    if (dtype != SF_DTYPE_BF16 && dtype != SF_DTYPE_F16 && dtype != SF_DTYPE_F32) return SF_EDTYPE;
    if (a.rows >= (size_t(1) << 31) || a.ld < a.vocab) return SF_EINVAL;
    if (misaligned(a.logits, dtype == SF_DTYPE_F32 ? 4 : 2) || misaligned(work, 16)) return SF_EALIGN;
    return SF_OK;
}

int dispatch_rows(Rows a, int dtype, void* work, bool top, hipStream_t st) {
    const Plan p = plan_of(a.vocab, dtype);
    const uint64_t most = rows_at_once(p), held = a.rows < most ? a.rows : most;
    a.parts = p.parts, a.per = p.per, a.list = p.list;
    a.part = static_cast<Part*>(work);
    a.lists = reinterpret_cast<uint64_t*>(a.part + held * p.parts);
    if (dtype == SF_DTYPE_BF16) return run_rows<Bf16>(a, p, top, st);
    if (dtype == SF_DTYPE_F16) return run_rows<F16>(a, p, top, st);
    return run_rows<F32>(a, p, top, st);
}

}  // namespace

extern "C" {

size_t sf_rows_work(size_t rows, size_t vocab, int dtype) {
    if (rows == 0 || vocab == 0 || vocab > (size_t(1) << 30)) return 0;
    const Plan p = plan_of(vocab, dtype);
    const uint64_t most = rows_at_once(p);
    return (rows < most ? rows : most) * p.parts * (sizeof(Part) + 8 * size_t(p.list));
}

int sf_top_logps(const void* logits, int dtype, size_t ld, size_t rows, size_t vocab, int k, double temperature, void* work,
                 float* logps, int64_t* ids, sf_stream_t stream) {
    if (rows == 0) return SF_OK;
    if (vocab == 0 || vocab > (size_t(1) << 30) || k < 1 || k > int(kMost) || size_t(k) > vocab || !(temperature > 0.0))
        return SF_EINVAL;
    Rows a = {};
    a.logits = logits, a.ld = ld, a.rows = rows, a.vocab = uint32_t(vocab);
    a.temperature = temperature, a.top_p = 1.0, a.top_k = k;
    a.logps = logps, a.ids = ids;
    const int e = check_rows(a, dtype, work);
    return e != SF_OK ? e : dispatch_rows(a, dtype, work, true, reinterpret_cast<hipStream_t>(stream));
}

int sf_sample_tokens(const void* logits, int dtype, size_t ld, size_t rows, size_t vocab, const float* uniforms,
                     double temperature, const float* temperatures, int64_t top_k, const int64_t* top_ks, double top_p,
                     const float* top_ps, double min_p, const float* min_ps, void* work, int64_t* ids, float* logps,
                     sf_stream_t stream) {
    if (rows == 0) return SF_OK;
    if (vocab == 0 || vocab > (size_t(1) << 30) || uniforms == nullptr) return SF_EINVAL;
    Rows a = {};
    a.logits = logits, a.ld = ld, a.rows = rows, a.vocab = uint32_t(vocab);
    a.temperature = temperature, a.temperatures = temperatures, a.top_k = top_k, a.top_ks = top_ks;
    a.top_p = top_p, a.top_ps = top_ps, a.min_p = min_p, a.min_ps = min_ps;
    a.uniforms = uniforms, a.logps = logps, a.ids = ids;
    const int e = check_rows(a, dtype, work);
    return e != SF_OK ? e : dispatch_rows(a, dtype, work, false, reinterpret_cast<hipStream_t>(stream));
}

}  // extern "C"
