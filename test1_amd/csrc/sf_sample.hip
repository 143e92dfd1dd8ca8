// The largest log-probabilities of rows of logits, and one token drawn from each
// row after temperature, top-k, top-p and min-p, for MI355X (gfx950).
//
// Words are ordered by falling logit, the first of equals first.  With w_j =
// exp((x_j - max) / T) a row keeps a prefix of that order: the first top_k; of
// those the words with less than top_p of their mass before them; of those the
// words with w_j >= min_p.  The word drawn is the first kept one, by its index,
// whose running mass exceeds u times the kept mass: no sort of the vocabulary.
// Which word that is hangs on sums of up to 2^30 terms, so masses are 64-bit.
//
// Two launches.  rows_parts_kernel cuts rows into parts of up to 2048 16-byte
// vectors, which a workgroup holds in registers, and leaves of each its maximum,
// its mass relative to that, and what the row's border will need: the words that
// may be among the k largest of it, or a histogram of its masses.  The chip is
// filled by parts, whatever the rows.  A workgroup for each row then joins its
// parts and finds the border and the word, reading again what it needs.  Rows
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
constexpr uint32_t kList = 512;           // candidates of a part, of a row's only part twice as many
constexpr uint32_t kBins = 256;           // of a part's histogram, T / kBinsOfT of logit each
constexpr float kBinsOfT = 16.0f;
constexpr uint32_t kSorted = 4096;        // candidates that a row sorts in LDS
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

// 2^y for y <= 0 or so: 2^n times the series of e^(f ln 2) to its 11th power, off
// by 6e-15 of itself.
struct Series {
    double c[12];
    constexpr Series() : c() {
        c[0] = 1.0;
        for (int i = 1; i < 12; ++i) c[i] = c[i - 1] * 0.69314718055994530941723212145818 / i;
    }
};
__constant__ constexpr Series kSeries{};
__device__ __forceinline__ double exp2_wide(double y) {
    y = fmax(y, -1100.0);
    const double n = rint(y), f = y - n;
    double p = kSeries.c[11];
#pragma unroll
    for (int i = 10; i >= 0; --i) p = fma(p, f, kSeries.c[i]);
    return ldexp(p, int(n));
}

// A row's vectors: whole 16-byte ones, its first and last may lie partly outside
// and are then read by elements, -inf where they are not the row's.
template <typename E>
struct Row {
    const Item<E>* x;
    uint32_t vocab, shift, vectors;   // the row begins `shift` elements into vector 0
    __device__ Row(const void* logits, uint64_t ld, uint64_t row, uint32_t vocab_) : vocab(vocab_) {
        x = static_cast<const Item<E>*>(logits) + row * ld;
        shift = uint32_t(reinterpret_cast<uintptr_t>(x) % 16) / sizeof(Item<E>);
        vectors = (vocab + shift + kOf<E> - 1) / kOf<E>;
    }
    __device__ u32x4 load(uint32_t v) const {
        const int64_t at = int64_t(v) * kOf<E> - shift;
        if (at >= 0 && at + kOf<E> <= vocab) return *reinterpret_cast<const u32x4*>(x + at);
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
    __device__ uint32_t index(uint32_t v, uint32_t i) const { return v * kOf<E> + i - shift; }
};
template <typename E>
__device__ __forceinline__ u32x4 nothing() {
    const uint32_t w = std::is_same_v<E, F32> ? 0xFF800000u : std::is_same_v<E, Bf16> ? Bf16::kNegInf2 : F16::kNegInf2;
    return u32x4{w, w, w, w};
}

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
    uint64_t* lists;            // [rows, parts, list]: places, or masses and counts of bins
    // settings: of all rows, or of each
    double temperature, top_p, min_p;
    int64_t top_k;
    const float *temperatures, *top_ps, *min_ps;
    const int64_t* top_ks;
    bool top_only;              // no draw: the k largest
    float* logps;
    int64_t* ids;
    const float* uniforms;
};

struct Settings {
    double t, top_p, min_p;
    uint32_t k;       // vocab: every word
    bool listed;      // by the parts' lists, else by masses
    bool filtered;    // of the latter: not every word is kept
    bool bins;        // of those: a border to find
};
__device__ __forceinline__ Settings settings(const Rows& a, uint64_t row) {
    Settings s;
    s.t = a.temperatures != nullptr ? double(a.temperatures[row]) : a.temperature;
    s.top_p = a.top_ps != nullptr ? double(a.top_ps[row]) : a.top_p;
    s.min_p = a.min_ps != nullptr ? double(a.min_ps[row]) : a.min_p;
    const int64_t k = a.top_ks != nullptr ? a.top_ks[row] : a.top_k;
    s.k = k <= 0 || k >= int64_t(a.vocab) ? a.vocab : uint32_t(k);
    if (!(s.t > 0.0)) s.t = 1.0, s.k = 1;   // the largest
    s.t = fmin(fmax(s.t, 1e-30), 1e30);     // so that neither it nor its inverse is infinite in fp32
    s.listed = a.top_only || s.k <= kMost;
    if (a.top_only) s.k = uint32_t(a.top_k);
    s.bins = s.top_p < 1.0 || s.k < a.vocab;
    s.filtered = s.bins || s.min_p > 0.0;
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
template <typename E, uint32_t kV>
__global__ __launch_bounds__(kPartLanes) void rows_parts_kernel(const Rows a) {
    constexpr uint32_t kN = kOf<E>;
    __shared__ float shared_m[kPartLanes / 64];
    __shared__ double shared_s[kPartLanes / 64];
    __shared__ uint32_t count;
    __shared__ float bound_of;
    __shared__ uint64_t mass[kBins];
    __shared__ uint32_t number[kBins];
    float* const most = reinterpret_cast<float*>(mass);   // [kPartLanes]
    const uint64_t row = blockIdx.x / a.parts;
    const uint32_t part = blockIdx.x % a.parts;
    const Settings s = settings(a, a.first + row);
    const Row<E> r(a.logits, a.ld, a.first + row, a.vocab);
    u32x4 x[kV];
#pragma unroll
    for (uint32_t i = 0; i < kV; ++i) {
        const uint32_t in = i * kPartLanes + threadIdx.x, v = part * a.per + in;
        x[i] = in < a.per && v < r.vectors ? r.load(v) : nothing<E>();
    }
    float mine = kNegInf;
#pragma unroll
    for (uint32_t i = 0; i < kV; ++i)
#pragma unroll
        for (uint32_t j = 0; j < kN; ++j) mine = fmaxf(mine, item<E>(x[i], j));
    if (threadIdx.x == 0) count = 0;
    const float m = block_all<kPartLanes>(mine, shared_m, Max{});
    Part* const out = a.part + row * a.parts + part;
    uint64_t* const list = a.lists + (row * a.parts + part) * a.list;
    const float from = base(m);

    if (s.listed) {
        const float c = float(double(kLog2e) / s.t);
        float sum = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < kV; ++i)
#pragma unroll
            for (uint32_t j = 0; j < kN; ++j) sum += __builtin_amdgcn_exp2f((item<E>(x[i], j) - from) * c);
        // A bound with k words of the part or more above it: the k-th largest of the
        // lanes' maxima, to 16 bits.  Of 256 lanes about 256 ln(256 / (256 - k)) words are.
        most[threadIdx.x] = mine;
        const double total = block_all<kPartLanes>(double(sum), shared_s, Add{});
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
            }
            if (threadIdx.x == 0) bound_of = float_of(bound << 16);
        }
        __syncthreads();
        const float bound = bound_of;
        // a bound of NaN's bits is that of fewer lanes than k: every word
        if (mine >= bound || bound != bound)
#pragma unroll
            for (uint32_t i = 0; i < kV; ++i)
#pragma unroll
                for (uint32_t j = 0; j < kN; ++j) {
                    const float f = item<E>(x[i], j);
                    if (f > kNegInf && !(f < bound)) {
                        const uint32_t at = atomicAdd(&count, 1u);
                        if (at < a.list) list[at] = place_of(f, r.index(part * a.per + i * kPartLanes + threadIdx.x, j));
                    }
                }
        __syncthreads();
        if (threadIdx.x == 0) *out = Part{m, count, total};
        return;
    }
    const double c = 1.4426950408889634073599 / s.t;
    const float scale = bin_scale(s.t), top_bin = floorf(m * scale);
    if (s.bins) {
        mass[threadIdx.x] = 0, number[threadIdx.x] = 0;
        __syncthreads();
    }
    // a part has at most 2^14 words: whole numbers of 2^-48
    double sum = 0.0;
    bool nan = false;
#pragma unroll
    for (uint32_t i = 0; i < kV; ++i)
#pragma unroll
        for (uint32_t j = 0; j < kN; ++j) {
            const float f = item<E>(x[i], j);
            nan |= f != f;
            const double w = exp2_wide((double(f) - double(from)) * c);
            sum += w;
            if (s.bins) {
                const float bin = top_bin - floorf(f * scale);
                if (bin >= 0.0f && bin < float(kBins)) {
                    atomicAdd(reinterpret_cast<unsigned long long*>(&mass[uint32_t(bin)]),
                              static_cast<unsigned long long>(w * 0x1p48 + 0.5));
                    atomicAdd(&number[uint32_t(bin)], 1u);
                }
            }
        }
    if (nan) sum = __builtin_nan("");
    sum = block_all<kPartLanes>(sum, shared_s, Add{});
    if (s.bins) {
        static_assert(kBins + kBins / 2 <= kList, "a list holds them");
        list[threadIdx.x] = mass[threadIdx.x];
        reinterpret_cast<uint32_t*>(list + kBins)[threadIdx.x] = number[threadIdx.x];
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
template <uint32_t kT>
__device__ Joined join_parts(const Rows& a, const Part* part, double c, double* shared) {
    float m = kNegInf;
    for (uint32_t p = threadIdx.x; p < a.parts; p += kT) m = fmaxf(m, part[p].m);
    m = block_all<kT>(m, reinterpret_cast<float*>(shared), Max{});
    if (__builtin_isinf(m)) return {m, 0.0, true};
    double sum = 0.0;
    for (uint32_t p = threadIdx.x; p < a.parts; p += kT)
        if (part[p].m > kNegInf || part[p].sum != part[p].sum) sum += part[p].sum * exp2_wide((double(part[p].m) - double(m)) * c);
    sum = block_all<kT>(sum, shared, Add{});
    return {m, sum, !(sum > 0.0)};
}

// places[0 .. n), n a power of two, by falling place.
template <uint32_t kT>
__device__ void sort_places(uint64_t* places, uint32_t n) {
    for (uint32_t size = 2; size <= n; size <<= 1)
        for (uint32_t d = size >> 1; d > 0; d >>= 1) {
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < n / 2; i += kT) {
                const uint32_t lo = (i & ~(d - 1)) << 1 | (i & (d - 1)), hi = lo | d;
                const uint64_t u = places[lo], v = places[hi];
                if ((u < v) == ((lo & size) == 0)) places[lo] = v, places[hi] = u;
            }
        }
    __syncthreads();
}
template <uint32_t kT>
__device__ uint32_t sort_padded(uint64_t* places, uint32_t n) {
    uint32_t pad = 2;
    while (pad < n) pad <<= 1;
    for (uint32_t i = n + threadIdx.x; i < pad; i += kT) places[i] = 0;
    sort_places<kT>(places, pad);
    return pad;
}

// What a row's workgroup has in LDS.
struct Shared {
    union {
        uint64_t places[kSorted];
        struct {
            uint64_t mass[2048];
            uint32_t number[2048];
        } digits;
        struct {
            uint64_t mass[kBins];
            uint32_t number[kBins];
        } bins;
    };
    double waves[16];
    double weights[kMost];
    uint32_t count, found_index;
    uint64_t found;
    double found_mass;
    uint32_t found_count, tied;
};

// The bin, of kN in falling order, in which a running count or mass first comes to `reach`,
// `before` of it ahead of all bins; kN where none does.  Left in sh with what comes before it
// and its number of words.
template <uint32_t kT, uint32_t kN>
__device__ void find_bin(const uint64_t* mass, const uint32_t* number, bool by_mass, uint64_t reach, uint64_t before_mass,
                         uint32_t before, Shared& sh) {
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
    uint64_t* const waves_m = reinterpret_cast<uint64_t*>(sh.waves);
    uint32_t* const waves_n = reinterpret_cast<uint32_t*>(sh.weights);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) waves_m[threadIdx.x >> 6] = upto_m, waves_n[threadIdx.x >> 6] = upto_n;
    if (threadIdx.x == 0) sh.found_index = kN;
    __syncthreads();
    uint64_t at_m = before_mass + upto_m - m;
    uint32_t at_n = upto_n - n;   // of these bins
    for (uint32_t w = 0; w < threadIdx.x >> 6; ++w) at_m += waves_m[w], at_n += waves_n[w];
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

// The words of a row in the order of their index: what `weight` (0: not taken) gives is
// added up, and the first word that takes the sum above `target` is found; where rounding
// leaves none, the last with a weight.  Every wave has a run of the row's vectors from v0
// to v1.  share: the target is that of the whole sum.
template <typename E, uint32_t kT, typename Weight>
__device__ uint32_t find_word(const Row<E>& r, uint32_t v0, uint32_t v1, double target, bool share, Weight weight, Shared& sh) {
    constexpr uint32_t kWaves = kT / 64;
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const uint32_t each = (v1 - v0 + kWaves - 1) / kWaves;
    const uint32_t from = min(v0 + wave * each, v1), to = min(from + each, v1);
    double sum = 0.0;
    uint32_t last = 0;   // index + 1 of the last with a weight
    for (uint32_t v = from + lane; v < to; v += 256) {
        u32x4 x[4];
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u) x[u] = v + u * 64 < to ? r.load(v + u * 64) : nothing<E>();
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u)
#pragma unroll
            for (uint32_t j = 0; j < kOf<E>; ++j) {
                const uint32_t index = r.index(v + u * 64, j);
                const double w = weight(item<E>(x[u], j), index);
                if (w > 0.0) sum += w, last = index + 1;
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
        for (uint32_t v = from + lane; !whole && v - lane < to; v += 64) {
            const u32x4 x = v < to ? r.load(v) : nothing<E>();
            double own = 0.0;
#pragma unroll
            for (uint32_t j = 0; j < kOf<E>; ++j) own += weight(item<E>(x, j), r.index(v, j));
            double upto = own;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const double below = __shfl_up(upto, d);
                if (lane >= uint32_t(d)) upto += below;
            }
            const uint64_t over = __ballot(upto > rest && own > 0.0);
            if (over != 0) {
                const uint32_t at = __ffsll(static_cast<unsigned long long>(over)) - 1;
                if (lane == at) {
                    double c = upto - own;
                    uint32_t pick = 0;
#pragma unroll
                    for (uint32_t j = 0; j < kOf<E>; ++j) {
                        const double w = weight(item<E>(x, j), r.index(v, j));
                        if (w > 0.0 && (pick == 0 || c <= rest)) pick = r.index(v, j) + 1;
                        c += w;
                    }
                    sh.found_index = pick;
                }
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
    for (uint32_t v = threadIdx.x; v < r.vectors; v += kT * 4) {
        u32x4 x[4];
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u) x[u] = v + u * kT < r.vectors ? r.load(v + u * kT) : nothing<E>();
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u)
#pragma unroll
            for (uint32_t j = 0; j < kOf<E>; ++j) f(item<E>(x[u], j), r.index(v + u * kT, j));
    }
}

// The border of a row by three passes over the digits of its words' keys: the place of the last
// word of the prefix that a count (so many words) or a mass (the words with less than `reach`
// before them) asks for, 0 for every word.  prefix_mass: of the prefix, or null.
template <typename E, uint32_t kT>
__device__ uint64_t border_by_digits(const Row<E>& r, float m, double c, bool by_mass, double reach, double* prefix_mass,
                                     Shared& sh) {
    // masses in whole numbers whose sum 62 bits hold
    const int bits = 62 - (32 - __builtin_clz(r.vocab));
    const double one = ldexp(1.0, bits);
    const auto whole = [&](float f) { return uint64_t(exp2_wide((double(f) - double(m)) * c) * one + 0.5); };
    const uint64_t target = by_mass ? uint64_t(ceil(fmax(reach, 0.0) * one)) : uint64_t(reach);
    uint32_t prefix = 0, known = 0, before = 0;
    uint64_t before_mass = 0;
    for (int pass = 0; pass < 3; ++pass) {
        const uint32_t width = pass < 2 ? 11 : 10, left = 32 - known - width;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < 2048; i += kT) sh.digits.mass[i] = 0, sh.digits.number[i] = 0;
        __syncthreads();
        each_word<E, kT>(r, [&](float f, uint32_t) {
            if (!(f > kNegInf)) return;
            const uint32_t key = key_of(f);
            if (known > 0 && (key >> (32 - known)) != prefix) return;
            const uint32_t bin = 2047 - ((key >> left) & ((1u << width) - 1));   // falling
            atomicAdd(&sh.digits.number[bin], 1u);
            atomicAdd(reinterpret_cast<unsigned long long*>(&sh.digits.mass[bin]), static_cast<unsigned long long>(whole(f)));
        });
        __syncthreads();
        find_bin<kT, 2048>(sh.digits.mass, sh.digits.number, by_mass, target, before_mass, before, sh);
        const uint32_t bin = sh.found_index;
        if (bin == 2048) return 0;   // the row has less
        prefix = prefix << width | ((2047 - bin) & ((1u << width) - 1));
        known += width;
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
    const uint32_t index = find_word<E, kT>(
        r, 0, r.vectors, double(take) - 0.5, false, [&](float f, uint32_t) { return f > kNegInf && key_of(f) == prefix ? 1.0 : 0.0; }, sh);
    return uint64_t(prefix) << 32 | uint32_t(~index);
}

// The same from the parts' histograms: the bin with the border, whose words are sorted.
// false: what is looked for lies below them, or the bin holds too many.
template <typename E, uint32_t kT>
__device__ bool border_by_bins(const Rows& a, const Part* part, const uint64_t* lists, const Row<E>& r, float m, double t,
                               bool by_mass, double reach, uint64_t* border, double* prefix_mass, Shared& sh) {
    const double c = 1.4426950408889634073599 / t;
    const float scale = bin_scale(t), top_bin = floorf(m * scale);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < kBins; i += kT) sh.bins.mass[i] = 0, sh.bins.number[i] = 0;
    __syncthreads();
    if (!(fabsf(top_bin) < 0x1p23f)) return false;   // bins that floats do not tell apart
    // 2^-44 of the largest weight: a row of up to 2^18 words; longer ones by digits
    if (r.vocab > (1u << 18)) return false;
    for (uint32_t i = threadIdx.x; i < a.parts * kBins; i += kT) {
        const uint32_t p = i / kBins, bin = i % kBins;
        if (!(part[p].m > kNegInf)) continue;
        const float offset = top_bin - floorf(part[p].m * scale) + float(bin);
        const uint32_t number = reinterpret_cast<const uint32_t*>(lists + uint64_t(p) * a.list + kBins)[bin];
        if (number == 0 || !(offset < float(kBins))) continue;
        const double by = exp2_wide((double(part[p].m) - double(m)) * c) * 0x1p-4;
        atomicAdd(&sh.bins.number[uint32_t(offset)], number);
        atomicAdd(reinterpret_cast<unsigned long long*>(&sh.bins.mass[uint32_t(offset)]),
                  static_cast<unsigned long long>(double(lists[uint64_t(p) * a.list + bin]) * by + 0.5));
    }
    __syncthreads();
    find_bin<kT, kBins>(sh.bins.mass, sh.bins.number, by_mass,
                        by_mass ? uint64_t(ceil(fmax(reach, 0.0) * 0x1p44)) : uint64_t(reach), 0, 0, sh);
    const uint32_t bin = sh.found_index, n = sh.tied, before = sh.found_count;
    const double before_mass = double(sh.found) * 0x1p-44;
    if (bin == kBins || n > kSorted) return false;
    __syncthreads();
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    each_word<E, kT>(r, [&](float f, uint32_t index) {
        if (f > kNegInf && top_bin - floorf(f * scale) == float(bin)) {
            const uint32_t at = atomicAdd(&sh.count, 1u);
            if (at < kSorted) sh.places[at] = place_of(f, index);
        }
    });
    __syncthreads();
    if (sh.count != n) return false;
    sort_padded<kT>(sh.places, n);
    // one wave along the sorted words, 64 at a time
    if (threadIdx.x < 64) {
        double before_here = before_mass;
        uint64_t last = 0;
        double mass = 0.0;
        for (uint32_t i0 = 0; i0 < n; i0 += 64) {
            const uint32_t i = i0 + threadIdx.x;
            const uint64_t place = i < n ? sh.places[i] : 0;
            const double w = i < n ? exp2_wide((double(logit_of(place)) - double(m)) * c) : 0.0;
            double upto = w;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const double below = __shfl_up(upto, d);
                if (threadIdx.x >= uint32_t(d)) upto += below;
            }
            const bool in = i < n && (by_mass ? before_here + (upto - w) < reach || (before + i == 0) : double(before + i) < reach);
            const uint64_t took = __ballot(in);
            if (took == 0) break;
            const int end = 63 - __builtin_clzll(took);
            last = __shfl(place, end);
            mass = before_here + __shfl(upto, end);
            before_here += __shfl(upto, 63);
        }
        if (threadIdx.x == 0) sh.found = last, sh.found_mass = mass;
    }
    __syncthreads();
    // a bin is reached before its first word where masses were rounded: then that is the border
    *border = sh.found != 0 ? sh.found : sh.places[0];
    if (prefix_mass != nullptr) *prefix_mass = sh.found_mass;
    __syncthreads();
    return true;
}

// The words of the parts' lists, sorted in sh.places; their number, or kSorted + 1 where a list
// or this one did not hold them.
template <uint32_t kT>
__device__ uint32_t sorted_lists(const Rows& a, const Part* part, const uint64_t* lists, Shared& sh) {
    __syncthreads();
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    for (uint32_t p = threadIdx.x / 64; p < a.parts; p += kT / 64) {
        const uint32_t n = part[p].count;
        uint32_t at = 0;
        if ((threadIdx.x & 63) == 0) at = atomicAdd(&sh.count, n <= a.list ? n : kSorted + 1);
        at = __shfl(at, 0);
        for (uint32_t i = threadIdx.x & 63; i < min(n, a.list); i += 64)
            if (at + i < kSorted) sh.places[at + i] = lists[uint64_t(p) * a.list + i];
        if (at > kSorted) break;
    }
    __syncthreads();
    const uint32_t n = sh.count;
    if (n > kSorted) return kSorted + 1;
    sort_padded<kT>(sh.places, n);
    return n;
}

// The k largest words of a row, sorted in sh.places, by whatever finds them; how many there are
// (-inf are none).
template <typename E, uint32_t kT>
__device__ uint32_t largest(const Rows& a, const Part* part, const uint64_t* lists, const Row<E>& r, float m, double c, uint32_t k,
                            Shared& sh) {
    uint32_t n = sorted_lists<kT>(a, part, lists, sh);
    if (n <= kSorted) return min(n, k);
    const uint64_t border = border_by_digits<E, kT>(r, m, c, false, double(k), nullptr, sh);
    __syncthreads();
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    each_word<E, kT>(r, [&](float f, uint32_t index) {
        if (f > kNegInf && place_of(f, index) >= border) {
            const uint32_t at = atomicAdd(&sh.count, 1u);
            if (at < kSorted) sh.places[at] = place_of(f, index);
        }
    });
    __syncthreads();
    n = min(sh.count, kSorted);
    sort_padded<kT>(sh.places, n);
    return min(n, k);
}

constexpr uint32_t kTopLanes = 256;
template <typename E>
__global__ __launch_bounds__(kTopLanes) void top_rows_kernel(const Rows a) {
    __shared__ Shared sh;
    const uint64_t row = blockIdx.x, of = a.first + row;
    const Part* const part = a.part + row * a.parts;
    const uint64_t* const lists = a.lists + row * a.parts * a.list;
    const Settings s = settings(a, of);
    const double c = 1.4426950408889634073599 / s.t;
    const Joined j = join_parts<kTopLanes>(a, part, c, sh.waves);
    float* const logps = a.logps + of * s.k;
    int64_t* const ids = a.ids + of * s.k;
    if (j.bad) {
        for (uint32_t i = threadIdx.x; i < s.k; i += kTopLanes) logps[i] = __builtin_nanf(""), ids[i] = -1;
        return;
    }
    const Row<E> r(a.logits, a.ld, of, a.vocab);
    const uint32_t n = largest<E, kTopLanes>(a, part, lists, r, j.m, c, s.k, sh);
    const double lse = log(j.sum);
    for (uint32_t i = threadIdx.x; i < n; i += kTopLanes) {
        logps[i] = float((double(logit_of(sh.places[i])) - double(j.m)) / s.t - lse);
        ids[i] = index_of(sh.places[i]);
    }
    // words of probability 0 in the order of their index
    for (uint32_t done = n, v0 = 0; done < s.k; v0 += kTopLanes) {
        uint32_t found = 0;
        const uint32_t index = v0 + threadIdx.x;
        bool none = false;
        if (index < a.vocab) {
            if constexpr (std::is_same_v<E, F32>) none = r.x[index] == 0xFF800000u;
            else none = r.x[index] == E::kNegInf;
        }
        const uint64_t those = __ballot(none);
        uint32_t* const waves = reinterpret_cast<uint32_t*>(sh.waves);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = __popcll(those);
        __syncthreads();
        uint32_t at = done + __popcll(those & ((uint64_t(1) << (threadIdx.x & 63)) - 1));
        for (uint32_t w = 0; w < kTopLanes / 64; ++w) {
            if (w < threadIdx.x >> 6) at += waves[w];
            found += waves[w];
        }
        if (none && at < s.k) logps[at] = kNegInf, ids[at] = index;
        done += found;
        if (v0 >= a.vocab) break;
    }
}

constexpr uint32_t kDrawLanes = 1024;
template <typename E>
__global__ __launch_bounds__(kDrawLanes) void draw_rows_kernel(const Rows a) {
    __shared__ Shared sh;
    const uint64_t row = blockIdx.x, of = a.first + row;
    const Part* const part = a.part + row * a.parts;
    const uint64_t* const lists = a.lists + row * a.parts * a.list;
    const Settings s = settings(a, of);
    const double c = 1.4426950408889634073599 / s.t;
    const Joined j = join_parts<kDrawLanes>(a, part, c, sh.waves);
    if (j.bad) {
        if (threadIdx.x == 0) a.ids[of] = -1, a.logps[of] = __builtin_nanf("");
        return;
    }
    const Row<E> r(a.logits, a.ld, of, a.vocab);
    // a share of the mass below 1; what is no number is 0
    float u = a.uniforms[of];
    u = u > 0.0f ? fminf(u, 0x1.fffffep-1f) : 0.0f;
    const double least = s.min_p > 0.0 ? fmin(log(s.min_p), 0.0) * s.t : -__builtin_inf();   // of x - max
    const double lse = log(j.sum);

    if (s.listed) {
        const uint32_t n = largest<E, kDrawLanes>(a, part, lists, r, j.m, c, s.k, sh);
        // n <= kMost words, one each for the first lanes
        const bool mine = threadIdx.x < n;
        const uint64_t place = mine ? sh.places[threadIdx.x] : 0;
        const double d = mine ? double(logit_of(place)) - double(j.m) : 0.0, w = mine ? exp2_wide(d * c) : 0.0;
        if (mine) sh.weights[threadIdx.x] = w;
        __syncthreads();
        double before = 0.0, total = 0.0;
        if (mine)
            for (uint32_t i = 0; i < n; ++i) {
                if (i == threadIdx.x) before = total;
                total += sh.weights[i];
            }
        const bool kept = mine && (!(s.top_p < 1.0) || threadIdx.x == 0 || before < s.top_p * total) && d >= least;
        __syncthreads();
        if (mine) sh.weights[threadIdx.x] = kept ? w : 0.0;
        if (threadIdx.x == 0) sh.found = 0;
        __syncthreads();
        if (kept && w > 0.0) {
            const uint32_t index = index_of(place);
            double mass = 0.0, upto = 0.0;
            for (uint32_t i = 0; i < n; ++i) {
                const double v = sh.weights[i];
                mass += v;
                if (index_of(sh.places[i]) <= index) upto += v;
            }
            // the first word above the target; where rounding leaves none, the last
            const bool over = upto > double(u) * mass;
            atomicMax(reinterpret_cast<unsigned long long*>(&sh.found),
                      uint64_t(over) << 63 | uint64_t(over ? ~index : index) << 16 | threadIdx.x);
        }
        __syncthreads();
        const uint32_t chosen = uint32_t(sh.found & 0xFFFF);
        if (threadIdx.x == chosen) a.ids[of] = index_of(place), a.logps[of] = float(d / s.t - lse);
        return;
    }
    uint32_t index;
    if (!s.filtered) {
        // the part, then the word within it
        const double target = double(u) * j.sum;
        double before = 0.0;
        uint32_t chosen = a.parts, fallback = 0;
        for (uint32_t p = 0; p < a.parts && chosen == a.parts; ++p) {
            if (!(part[p].m > kNegInf)) continue;
            const double mass = part[p].sum * exp2_wide((double(part[p].m) - double(j.m)) * c);
            if (mass > 0.0) fallback = p;
            if (before + mass > target) chosen = p;
            else before += mass;
        }
        const bool none = chosen == a.parts;
        if (none) chosen = fallback;
        const uint32_t v0 = min(chosen * a.per, r.vectors), v1 = min(v0 + a.per, r.vectors);
        index = find_word<E, kDrawLanes>(
            r, v0, v1, none ? __builtin_inf() : target - before, false,
            [&](float f, uint32_t) { return exp2_wide((double(f) - double(j.m)) * c); }, sh);
    } else {
        uint64_t border = 0;
        double mass = j.sum;
        if (s.k < a.vocab) {
            if (!border_by_bins<E, kDrawLanes>(a, part, lists, r, j.m, s.t, false, double(s.k), &border, &mass, sh))
                border = border_by_digits<E, kDrawLanes>(r, j.m, c, false, double(s.k), &mass, sh);
            if (border == 0) mass = j.sum;
        }
        if (s.top_p < 1.0) {
            const double reach = s.top_p * mass;
            uint64_t nucleus = 0;
            if (!border_by_bins<E, kDrawLanes>(a, part, lists, r, j.m, s.t, true, reach, &nucleus, nullptr, sh))
                nucleus = border_by_digits<E, kDrawLanes>(r, j.m, c, true, reach, nullptr, sh);
            border = max(border, nucleus);
        }
        index = find_word<E, kDrawLanes>(
            r, 0, r.vectors, double(u), true,
            [&](float f, uint32_t i) {
                const double d = double(f) - double(j.m);
                return f > kNegInf && d >= least && place_of(f, i) >= border ? exp2_wide(d * c) : 0.0;
            },
            sh);
    }
    if (threadIdx.x == 0) {
        index = min(index, a.vocab - 1);
        float f;
        if constexpr (std::is_same_v<E, F32>) f = __uint_as_float(r.x[index]);
        else f = E::lo(r.x[index]);
        a.ids[of] = index;
        a.logps[of] = float((double(f) - double(j.m)) / s.t - lse);
    }
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
// Rows of one pair of launches: 256 MiB of lists.
uint64_t rows_at_once(const Plan& p) {
    const uint64_t rows = (uint64_t(256) << 20) / (uint64_t(p.parts) * (8 * p.list + sizeof(Part)));
    return rows > 0 ? rows : 1;
}

template <typename E>
int launch_parts(const Rows& a, uint32_t rows, uint32_t lane, hipStream_t st) {
    const auto kernel = lane == 1   ? rows_parts_kernel<E, 1>
                        : lane == 2 ? rows_parts_kernel<E, 2>
                        : lane == 4 ? rows_parts_kernel<E, 4>
                                    : rows_parts_kernel<E, 8>;
    hipLaunchKernelGGL(kernel, dim3(rows * a.parts), dim3(kPartLanes), 0, st, a);
    return status();
}

template <typename E>
int run_rows(Rows a, const Plan& p, hipStream_t st) {
    const uint64_t most = rows_at_once(p);
    for (uint64_t r = 0; r < a.rows; r += most) {
        const uint32_t n = uint32_t(a.rows - r < most ? a.rows - r : most);
        a.first = r;
        int e = launch_parts<E>(a, n, p.lane, st);
        if (e != SF_OK) return e;
        if (a.top_only) hipLaunchKernelGGL(top_rows_kernel<E>, dim3(n), dim3(kTopLanes), 0, st, a);
        else hipLaunchKernelGGL(draw_rows_kernel<E>, dim3(n), dim3(kDrawLanes), 0, st, a);
        e = status();
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

int dispatch_rows(Rows a, int dtype, void* work, hipStream_t st) {
    const Plan p = plan_of(a.vocab, dtype);
    const uint64_t most = rows_at_once(p), held = a.rows < most ? a.rows : most;
    a.parts = p.parts, a.per = p.per, a.list = p.list;
    a.part = static_cast<Part*>(work);
    a.lists = reinterpret_cast<uint64_t*>(a.part + held * p.parts);
    if (dtype == SF_DTYPE_BF16) return run_rows<Bf16>(a, p, st);
    if (dtype == SF_DTYPE_F16) return run_rows<F16>(a, p, st);
    return run_rows<F32>(a, p, st);
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
    a.temperature = temperature, a.top_p = 1.0, a.top_k = k, a.top_only = true;
    a.logps = logps, a.ids = ids;
    const int e = check_rows(a, dtype, work);
    return e != SF_OK ? e : dispatch_rows(a, dtype, work, reinterpret_cast<hipStream_t>(stream));
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
    return e != SF_OK ? e : dispatch_rows(a, dtype, work, reinterpret_cast<hipStream_t>(stream));
}

}  // extern "C"
