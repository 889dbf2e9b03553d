// Sampling a token from a row of logits: temperature, top-k, top-p and min-p, with a given uniform number.
//
//   w_j = exp((z_j - max z) / T)                      (temperature)
//   order: logits descending, equal ones by index ascending
//   keep the first top_k                              (top-k)
//   of those keep each whose predecessors weigh less than top_p times all of them together   (top-p)
//   of those keep w_j >= min_p                        (min-p)
//   token = the first j, by index, at which the kept weights' running sum exceeds u times their sum.
// The first of the order is always kept.  -infinity and NaN are masked: never drawn, never counted.  T = 0 takes the
// first of the order.
//
// Which token is drawn is a comparison of a long sum with a border, so weights are 64-bit fixed point: exp in fp64,
// rounded once to a multiple of 2^-43 (2^20 classes of weight 1 sum to 2^63).  Integer sums have no order: histograms by
// LDS atomics and sums over waves in any order give the same token on every run.
//
// No row is sorted.  A cut of the order (top-k by counts, top-p by mass) is a border key (the order-preserving bits of
// the logits) and how many tokens of exactly that key stay, by index.  Rows of up to 1024 classes: 16 or 64
// lanes a row, the border by bisection of the key's bits.  Longer rows: one workgroup a row, in registers
// where they fit, with the paths below.
#include "tokens.hpp"

#include <cfloat>
#include <climits>
#include <cmath>

namespace rl {
namespace sample {

using tokens::Row;
using tokens::Team;

typedef unsigned long long u64;

constexpr int kMaxClasses = 1 << 20;
constexpr double kScale = 0x1p43;  // weight 1

struct Params {
    const void* logits;
    long long ld, rows;
    int classes;
    double temperature, top_p, min_p;      // where the arrays are null
    int top_k;
    const float *temperatures, *top_ps, *min_ps;
    const int* top_ks;
    const float* uniform;
    long long* tokens;
    float* log_probs;
};

// One row's settings.
struct Settings {
    double temperature, per_t, top_p;
    u64 min_weight;  // fixed point
    int top_k;
    float u;
    bool valid;

    __device__ __forceinline__ Settings(const Params& p, long long r) {
        temperature = p.temperatures ? p.temperatures[r] : p.temperature;
        top_p = p.top_ps ? p.top_ps[r] : p.top_p;
        const double min_p = p.min_ps ? p.min_ps[r] : p.min_p;
        top_k = p.top_ks ? p.top_ks[r] : p.top_k;
        u = p.uniform[r];
        valid = temperature >= 0.0 && temperature < INFINITY && top_p == top_p && min_p == min_p && u == u;
        per_t = temperature > 0.0 ? 1.0 / temperature : 0.0;
        min_weight = static_cast<u64>(ceil(fmax(fmin(min_p, 1.0), 0.0) * kScale));
    }
    // only the first of the order can stay
    __device__ __forceinline__ bool one() const { return temperature == 0.0 || top_p <= 0.0 || top_k == 1; }
    __device__ __forceinline__ double target(u64 total) const {
        return fmax(fmin(static_cast<double>(u), 1.0 - 0x1p-50), 0.0) * static_cast<double>(total);
    }
};

// Bits that order as the values do (NaN excluded, -0 as 0).
__device__ __forceinline__ unsigned ordered(float z) {
    const unsigned b = __float_as_uint(z + 0.0f);
    return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
// The logit whose ordered bits are `key`.
__device__ __forceinline__ float from_ordered(unsigned key) {
    return __uint_as_float(key ^ (key >> 31 ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ bool masked(float z) { return !(z > -INFINITY); }  // -infinity or NaN

// exp((z - m) / T) as a multiple of 2^-43.  With t = (z - m) 32 log2(e) / T = 32 e + i + f, |f| <= 1/2, it is 2^e times
// 2^(i / 32), from a table of 32 (one LDS bank pair each), times the Taylor sum of exp(f ln2 / 32) to the fifth order, which
// leaves (ln2 / 64)^6 / 720 = 2e-15 of it: 20 instructions where exp() takes about 45.
constexpr int kTable = 32;
__device__ __forceinline__ void fill_table(double* table) {
    if (threadIdx.x < kTable) table[threadIdx.x] = exp2(static_cast<double>(threadIdx.x) / kTable);
}
struct Weights {
    const double* table;
    float m;
    double per_step;  // 32 log2(e) / T
    bool alone;       // only m itself weighs anything: an infinite maximum, or 1 / T past the doubles

    __device__ __forceinline__ Weights(const double* table_, float m_, double per_t)
        : table(table_), m(m_), per_step(per_t * (kTable * 1.44269504088896340736)) {
        alone = !(m < INFINITY) || !(per_step < INFINITY);
    }

    template <int N>
    __device__ __forceinline__ void operator()(const float (&z)[N], u64 (&w)[N]) const {
        if (alone) {
#pragma unroll
            for (int e = 0; e < N; ++e) w[e] = z[e] == m ? 1ULL << 43 : 0;
            return;
        }
        constexpr double kRound = 0x1.8p52;  // added and taken off again: the nearest whole number, whose bits end the sum
        constexpr double kStep = 0.693147180559945309417 / kTable;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            double t = (static_cast<double>(z[e]) - static_cast<double>(m)) * per_step;
            t = __builtin_fmax(t, -46.0 * kTable);  // rounds to weight 0, as NaN does
            const double sum = t + kRound;
            const double f = t - (sum - kRound);
            const int n = static_cast<int>(__double_as_longlong(sum));
            double x = __builtin_fma(f, kStep * kStep * kStep * kStep * kStep / 120, kStep * kStep * kStep * kStep / 24);
            x = __builtin_fma(f, x, kStep * kStep * kStep / 6);
            x = __builtin_fma(f, x, kStep * kStep / 2);
            x = __builtin_fma(f, x, kStep);
            x = __builtin_fma(f, x, 1.0);
            x *= table[n & (kTable - 1)];
            // times 2^(n >> 5); x lies in [0.98, 2), the power above 2^-47
            const u64 power = static_cast<u64>(static_cast<unsigned>(n >> 5) << 20) << 32;
            x = __longlong_as_double(__double_as_longlong(x) + static_cast<long long>(power));
            // added to 2^9 a weight of [0, 1] is rounded to a multiple of 2^-43 in the sum's last bits
            w[e] = static_cast<u64>(__double_as_longlong(x + 512.0) - __double_as_longlong(512.0));
        }
    }
    __device__ __forceinline__ u64 operator()(float z) const {
        const float v[1] = {z};
        u64 w[1];
        (*this)(v, w);
        return w[0];
    }
};

template <int Control>
__device__ __forceinline__ int dpp32(int v) {
    return __builtin_amdgcn_update_dpp(0, v, Control, 0xF, 0xF, true);
}
template <int Control>
__device__ __forceinline__ u64 dpp64(u64 v) {
    const unsigned lo = dpp32<Control>(static_cast<int>(v)), hi = dpp32<Control>(static_cast<int>(v >> 32));
    return (static_cast<u64>(hi) << 32) | lo;
}
__device__ __forceinline__ u64 lane64(u64 v, int lane) {
    const unsigned lo = __builtin_amdgcn_readlane(static_cast<int>(v), lane);
    const unsigned hi = __builtin_amdgcn_readlane(static_cast<int>(v >> 32), lane);
    return (static_cast<u64>(hi) << 32) | lo;
}
// Sum over a wave, in every lane.
__device__ __forceinline__ u64 wave_total(u64 v) {
    v += dpp64<kDppXor1>(v);
    v += dpp64<kDppXor2>(v);
    v += dpp64<kDppHalfMirror>(v);
    v += dpp64<kDppMirror>(v);
    return (lane64(v, 0) + lane64(v, 16)) + (lane64(v, 32) + lane64(v, 48));
}
// Inclusive prefix sum over a wave: shifts by 1, 2, 4 and 8 inside the rows of 16 lanes, then the rows before.
__device__ __forceinline__ u64 wave_scan(u64 v) {
    v += dpp64<0x111>(v);
    v += dpp64<0x112>(v);
    v += dpp64<0x114>(v);
    v += dpp64<0x118>(v);
    const u64 a = lane64(v, 15), b = a + lane64(v, 31), c = b + lane64(v, 47);
    const int row = threadIdx.x % kWave / 16;
    return v + (row == 0 ? 0 : row == 1 ? a : row == 2 ? b : c);
}
__device__ __forceinline__ int wave_scan(int v) { return static_cast<int>(wave_scan(static_cast<u64>(v))); }
__device__ __forceinline__ int wave_total(int v) { return static_cast<int>(wave_total(static_cast<u64>(v))); }
__device__ __forceinline__ unsigned wave_min(unsigned v) {
#pragma unroll
    for (int by = 32; by > 0; by /= 2) v = min(v, static_cast<unsigned>(__shfl_xor(static_cast<int>(v), by, kWave)));
    return v;
}

// The least whole number that, rounded to a double, exceeds `target` (not negative, below 2^63): from 2^53 on half a step
// past it, which rounds up from an odd last bit only.
__device__ __forceinline__ u64 first_past(double target) {
    const u64 whole = static_cast<u64>(target);
    if (target < 0x1p53) return whole + 1;
    const u64 bits = static_cast<u64>(__double_as_longlong(target));
    const u64 half = 1ULL << (static_cast<int>(bits >> 52) - 1023 - 53);
    return whole + half + (bits & 1 ? 0 : 1);
}

__device__ __forceinline__ void nothing_drawn(const Params& p, long long r, bool valid) {
    p.tokens[r] = -1;
    if (p.log_probs) p.log_probs[r] = valid ? -INFINITY : NAN;
}
__device__ __forceinline__ void drawn(const Params& p, long long r, long long token, float z, float m, double per_t, u64 total) {
    p.tokens[r] = token;
    if (!p.log_probs) return;
    const double x = z == m ? 0.0 : (static_cast<double>(z) - static_cast<double>(m)) * per_t;
    p.log_probs[r] = static_cast<float>(x - log(static_cast<double>(total) / kScale));
}

// How many of the tokens of a border key stay (at most `ties`): the i-th does while the mass before it, above + i tie, is
// below the border.
__device__ __forceinline__ int ties_below(double border, u64 above, u64 tie, int ties) {
    const double stay = ceil((border - static_cast<double>(above)) / static_cast<double>(tie));
    return static_cast<int>(fmax(fmin(stay, static_cast<double>(ties)), 1.0));
}

// ---------------------------------------------------------------------------
// Up to 1024 classes: Lanes lanes a row (16: four rows a wave share its instructions), E consecutive classes a lane
// ---------------------------------------------------------------------------
// Bound by instructions, most of them the weights': 32768 x 256 bf16 without filters 12.9 us (23.9 with a wave a row; 14.8
// with comparisons in doubles, not whole numbers, to find the chosen class), greedy 9.0 us, with top-p 40 us (about 15
// bisection steps over all weights).
constexpr int kShortThreads = 256;

template <int Lanes>
struct Lane {
    static_assert(Lanes == 16 || Lanes == kWave, "a row of lanes or a wave");
    __device__ __forceinline__ static u64 total(u64 v) {
        if constexpr (Lanes == kWave) return wave_total(v);
        v += dpp64<kDppXor1>(v);
        v += dpp64<kDppXor2>(v);
        v += dpp64<kDppHalfMirror>(v);
        return v + dpp64<kDppMirror>(v);
    }
    __device__ __forceinline__ static u64 scan(u64 v) {
        if constexpr (Lanes == kWave) return wave_scan(v);
        v += dpp64<0x111>(v);
        v += dpp64<0x112>(v);
        v += dpp64<0x114>(v);
        return v + dpp64<0x118>(v);
    }
    __device__ __forceinline__ static int total(int v) {
        v += dpp32<kDppXor1>(v);
        v += dpp32<kDppXor2>(v);
        v += dpp32<kDppHalfMirror>(v);
        v += dpp32<kDppMirror>(v);
        if constexpr (Lanes == kWave)
            v = __builtin_amdgcn_readlane(v, 0) + __builtin_amdgcn_readlane(v, 16) + __builtin_amdgcn_readlane(v, 32) +
                __builtin_amdgcn_readlane(v, 48);
        return v;
    }
    __device__ __forceinline__ static int scan(int v) { return static_cast<int>(scan(static_cast<u64>(v))); }
    __device__ __forceinline__ static float max(float v) {
        if constexpr (Lanes == kWave) return wave_max(v);
        v = fmaxf(v, dpp<kDppXor1>(v));
        v = fmaxf(v, dpp<kDppXor2>(v));
        v = fmaxf(v, dpp<kDppHalfMirror>(v));
        return fmaxf(v, dpp<kDppMirror>(v));
    }
    __device__ __forceinline__ static unsigned max(unsigned v) {
        v = ::max(v, static_cast<unsigned>(dpp32<kDppXor1>(static_cast<int>(v))));
        v = ::max(v, static_cast<unsigned>(dpp32<kDppXor2>(static_cast<int>(v))));
        v = ::max(v, static_cast<unsigned>(dpp32<kDppHalfMirror>(static_cast<int>(v))));
        v = ::max(v, static_cast<unsigned>(dpp32<kDppMirror>(static_cast<int>(v))));
        if constexpr (Lanes == kWave) {
            const unsigned a = __builtin_amdgcn_readlane(v, 0), b = __builtin_amdgcn_readlane(v, 16);
            const unsigned c = __builtin_amdgcn_readlane(v, 32), d = __builtin_amdgcn_readlane(v, 48);
            v = ::max(::max(a, b), ::max(c, d));
        }
        return v;
    }
};

template <typename T, int Lanes, int E>
__global__ __launch_bounds__(kShortThreads) void sample_short(Params p) {
    typedef typename T::Store Store;
    typedef Lane<Lanes> L;
    constexpr int kRows = kShortThreads / Lanes;
    // the bits of a key that 16-bit logits cannot differ in are dropped: fewer to bisect
    constexpr int kShift = T::kKeyShift;
    __shared__ double table[kTable];
    fill_table(table);
    __syncthreads();
    const long long r = blockIdx.x * static_cast<long long>(kRows) + threadIdx.x / Lanes;
    if (r >= p.rows) return;
    const int lane = threadIdx.x % Lanes;
    const Settings s(p, r);
    const Store* row = static_cast<const Store*>(p.logits) + r * p.ld;
    const int first = lane * E;
    float z[E];
    if (first + E <= p.classes) {
        struct __attribute__((packed, aligned(sizeof(Store)))) Piece {
            Store v[E];
        };
        const Piece piece = *reinterpret_cast<const Piece*>(row + first);
#pragma unroll
        for (int e = 0; e < E; ++e) z[e] = T::value(piece.v[e]);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) z[e] = first + e < p.classes ? T::value(row[first + e]) : -INFINITY;
    }
    float m = -INFINITY;
#pragma unroll
    for (int e = 0; e < E; ++e) m = fmaxf(m, z[e]);
    m = L::max(m);
    if (!s.valid || m == -INFINITY) {
        if (lane == 0) nothing_drawn(p, r, s.valid);
        return;
    }
    if (s.one()) {
        unsigned back = 0;  // the first class of the maximum, counted from the end
#pragma unroll
        for (int e = 0; e < E; ++e) back = max(back, z[e] == m ? ~static_cast<unsigned>(first + e) : 0u);
        back = L::max(back);
        if (lane == 0) drawn(p, r, ~back, m, m, s.per_t, 1ULL << 43);
        return;
    }
    const Weights weight(table, m, s.per_t);
    u64 w[E];
    weight(z, w);
    if ((s.top_k > 0 && s.top_k < p.classes) || s.top_p < 1.0) {
        unsigned key[E];  // 0: masked
        const unsigned high = (ordered(m) >> kShift) + 1;
        unsigned far = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            key[e] = masked(z[e]) ? 0 : (ordered(z[e]) >> kShift) + 1;
            if (key[e]) far = max(far, high - key[e]);
        }
        const unsigned low = high - L::max(far);
        // (inlined by force: left as a call, one of these puts the row into scratch memory, 12.9 -> 18.3 us)
        // the largest key at which `reached` holds, which it does at `floor`; all keys lie in [low, high]
        const auto bisect = [&](unsigned floor, auto reached) __attribute__((always_inline)) {
            if (floor == high) return high;
            int bit = 31 - __clz(floor ^ high);
            unsigned border = high >> bit >> 1 << bit << 1;
            for (; bit >= 0; --bit)
                if (reached(border | (1u << bit))) border |= 1u << bit;
            return border;
        };
        const auto count_from = [&](unsigned k) __attribute__((always_inline)) {
            int n = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) n += key[e] >= k;
            return L::total(n);
        };
        const auto mass_from = [&](unsigned k) __attribute__((always_inline)) {
            u64 sum = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) sum += key[e] >= k ? w[e] : 0;
            return L::total(sum);
        };
        // what a token of key k weighs (the key occurs)
        const auto weight_at = [&](unsigned k) __attribute__((always_inline)) {
            unsigned lo = 0, hi = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                lo = key[e] == k ? static_cast<unsigned>(w[e]) : lo;
                hi = key[e] == k ? static_cast<unsigned>(w[e] >> 32) : hi;
            }
            return (static_cast<u64>(L::max(hi)) << 32) | L::max(lo);
        };
        unsigned border = 1;  // keys above it stay, and the first `ties` of those equal to it
        int ties = INT_MAX;
        if (s.top_k > 0 && s.top_k < count_from(1)) {
            border = bisect(low, [&](unsigned k) { return count_from(k) >= s.top_k; });
            ties = s.top_k - count_from(border + 1);
        }
        if (s.top_p < 1.0) {
            const bool limited = ties != INT_MAX;
            const u64 tie = limited ? weight_at(border) : 0;
            const u64 above = mass_from(limited ? border + 1 : 1);
            const double mass = s.top_p * static_cast<double>(above + (limited ? tie * static_cast<u64>(ties) : 0));
            if (static_cast<double>(above) >= mass) {
                border = bisect(max(border, low), [&](unsigned k) { return static_cast<double>(mass_from(k)) >= mass; });
                ties = ties_below(mass, mass_from(border + 1), weight_at(border), p.classes);
            } else if (tie > 0) {
                ties = ties_below(mass, above, tie, ties);
            }
        }
        int equal = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) equal += key[e] == border;
        int rank = L::scan(equal) - equal;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (key[e] < border || (key[e] == border && rank++ >= ties)) w[e] = 0;
    }
    if (s.min_weight) {
#pragma unroll
        for (int e = 0; e < E; ++e) w[e] = w[e] >= s.min_weight ? w[e] : 0;
    }
    u64 sum = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) sum += w[e];
    const u64 upto = L::scan(sum), total = L::total(sum);
    const u64 past = first_past(s.target(total));
    // the first lane that passes it is the one whose lanes before do not
    if (upto < past || upto - sum >= past) return;
    u64 run = upto - sum + w[0];
    int at = first;
    float chosen = z[0];
#pragma unroll
    for (int e = 1; e < E; ++e) {
        const bool further = run < past;
        at += further;
        chosen = further ? z[e] : chosen;
        run += w[e];
    }
    drawn(p, r, at, chosen, m, s.per_t, total);
}

// ---------------------------------------------------------------------------
// Longer rows: one workgroup a row
// ---------------------------------------------------------------------------
// 256 x 131072 bf16 (16 us to read at a copy's rate): greedy 21 us, top-k 64 with top-p 25 us, no filter 53 us, top-p alone 72
// to 102 us.  Where all of a row is weighed, the weights' instructions bound it: about 24 a class, 27 us a pass of 128
// classes a thread.  One row of 32768 fp32 with top-k and top-p: 12 us, a chain of 14 barriers.
constexpr int kBins = 1024;
constexpr int kBinsPerLane = kBins / kWave;
constexpr float kBinsPerUnit = 32.0f;  // linear bins of 1/32 of (max - z) / T: 32 units until the last one
constexpr int kDigit = 10;             // bits of a digit: a bin each
static_assert(kBins == 1 << kDigit, "a bin for each digit");
constexpr int kCandidates = 1024;
constexpr int kKept = 2048;
constexpr int kRanked = 128;      // candidates up to which counting the larger ones is faster than sorting

struct Ones {
    template <int N>
    __device__ __forceinline__ void operator()(const float (&)[N], u64 (&w)[N]) const {
#pragma unroll
        for (int e = 0; e < N; ++e) w[e] = 1;
    }
};

// The borders: a count, and a share of the sum, of which the sample's sum may be off.
struct CountBorder {
    int k;
    __device__ __forceinline__ double operator()(u64) const { return k; }
    __device__ __forceinline__ double slack(u64) const { return 0.5 * k + 16; }
};
struct ShareBorder {
    double share;
    u64 tied;  // what lies below the keys looked at and still counts
    __device__ __forceinline__ double operator()(u64 all) const { return share * static_cast<double>(all + tied); }
    __device__ __forceinline__ double slack(u64 all) const { return 0.03 * static_cast<double>(all); }
};

struct Shared {
    u64 bins[kBins];
    union {
        alignas(16) u64 list[kCandidates];  // candidates of top-k: key, then ~index
        struct {
            float value;
            int segment;
        } kept[kKept];
    };
    double table[kTable];
    u64 above;      // running sum before the bin found
    double border;
    int bin, count;
    unsigned low, high;
    float reduce[16];
    u64 sums[16], more_sums[16];
};

// Wave 0: the first bin, in order, at which the running sum reaches `border`; -1 if none does.  Leaves the sum before
// that bin (or of all) in `before`.
__device__ __forceinline__ int find_bin(const u64* bins, u64 start, double border, u64& before) {
    const int lane = threadIdx.x % kWave;
    u64 mine = 0;
#pragma unroll
    for (int i = 0; i < kBinsPerLane; ++i) mine += bins[lane * kBinsPerLane + i];
    const u64 upto = start + wave_scan(mine);
    const u64 found = __ballot(static_cast<double>(upto) >= border);
    if (!found) {
        before = lane64(upto, kWave - 1);
        return -1;
    }
    const int first = __ffsll(found) - 1;
    // the lane's bins, one a lane
    const u64 start_here = lane64(upto - mine, first);
    const u64 here = lane < kBinsPerLane ? bins[first * kBinsPerLane + lane] : 0;
    const u64 sum = start_here + wave_scan(here);
    const int at = __ffsll(__ballot(static_cast<double>(sum) >= border)) - 1;
    before = lane64(sum - here, at);
    return first * kBinsPerLane + at;
}

// The first key of [first, last] at which `reached` holds, as it does at `last` and from the first one on: 64 tries at a
// time by a wave.
template <typename F>
__device__ __forceinline__ unsigned first_key(unsigned first, unsigned last, F reached) {
    while (first < last) {
        const unsigned step = (last - first) / kWave + 1;
        const unsigned mine = min(first + (threadIdx.x % kWave) * step, last);
        const u64 votes = __ballot(reached(mine));
        const int lane = votes ? __ffsll(votes) - 1 : kWave;
        const unsigned start = first;
        if (lane > 0) first = min(start + (lane - 1) * step, last - 1) + 1;
        if (lane < kWave) last = min(start + lane * step, last);
    }
    return last;
}

template <typename T, int Group, bool Held>
struct Sampler {
    typedef Team<Group> G;
    typedef tokens::LongRow<T, Group, Held> R;
    static constexpr int V = T::kPerChunk;

    const R& row;
    Shared& s;
    const int t;
    const float m;         // the row's maximum
    const float per_bin;   // bins of a unit of logits
    int over_count = 0;    // how many values lay above the last cut's zone

    // Bins of 1 / scale from `origin` downwards; the last one takes all the rest.
    __device__ __forceinline__ static int bin_of(float z, float origin, float scale) {
        if (z == origin) return 0;
        const float d = (origin - z) * scale;
        return d < kBins - 1 ? static_cast<int>(d) : kBins - 1;
    }

    __device__ __forceinline__ void clear_bins() {
        for (int b = t; b < kBins; b += Group) s.bins[b] = 0;
        if (t == 0) {
            s.low = 0xffffffffu;
            s.high = 0;
            s.count = 0;
        }
        __syncthreads();
    }

    // Sums over the workgroup, in every thread.
    __device__ __forceinline__ void block_totals(u64& a, u64& b) {
        a = wave_total(a);
        b = wave_total(b);
        if (t % kWave == 0) {
            s.sums[t / kWave] = a;
            s.more_sums[t / kWave] = b;
        }
        __syncthreads();
        a = b = 0;
#pragma unroll
        for (int w = 0; w < G::kWaves; ++w) {
            a += s.sums[w];
            b += s.more_sums[w];
        }
    }

    // Where the border probably lies, from a sample: every thread's maximum (the heavy ones are among these), and the rest
    // of its first chunk for all its chunks.  Bins [from, to] of the distance to the maximum; false without a guess.
    template <typename F, typename B>
    __device__ __forceinline__ bool guess(F f, B border_of, float mine, int& from, int& to) {
        clear_bins();
        if (!masked(mine)) {
            const float one[1] = {mine};
            u64 w[1];
            f(one, w);
            atomicAdd(&s.bins[bin_of(mine, m, per_bin)], w[0]);
        }
        float v[V];
        u64 w[V];
        T::unpack(row.chunk(0), v);
        f(v, w);
        const u64 stands_for = static_cast<u64>(row.passes());
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (!masked(v[e]) && v[e] < mine) atomicAdd(&s.bins[bin_of(v[e], m, per_bin)], w[e] * stands_for);
        __syncthreads();
        if (t < kWave) {
            u64 all = 0, before;
#pragma unroll
            for (int i = 0; i < kBinsPerLane; ++i) all += s.bins[t * kBinsPerLane + i];
            all = wave_total(all);
            const double border = border_of(all), slack = border_of.slack(all);
            const int first = find_bin(s.bins, 0, fmax(border - slack, 0.0), before);
            const int last = find_bin(s.bins, 0, border + slack, before);
            if (t == 0) {
                s.bin = first;
                s.count = last < 0 ? kBins - 1 : last;
            }
        }
        __syncthreads();
        from = s.bin;
        to = s.count;
        return from >= 0;
    }

    // The key, above `floor`, at which the running sum of f reaches border_of(sum of all): in `key`, with the sum of
    // the keys above it in `above`.  False if none does; `above` is then the sum of all.  The border must be positive.
    //
    // One pass sums f over all keys and over those above a zone, and makes a histogram of those in it; a zone that came out
    // wrong is replaced by all keys.  Then digits of the keys in the bin in which the border lies, from the first bit in
    // which they can differ.  An atomic for every key would cost more than its weight: 131072 bf16, top-p alone, 151 us with
    // all keys for a zone.
    template <typename F, typename B>
    __device__ __forceinline__ bool cut_at(F f, B border_of, unsigned floor, float mine, unsigned& key, u64& above) {
        over_count = 0;
        const float under = floor ? from_ordered(floor) : -INFINITY;
        int from = 0, to = kBins - 1;
        if (!floor && row.passes() >= 4 && m < INFINITY && !guess(f, border_of, mine, from, to)) from = 0, to = kBins - 1;
        float origin, bottom, scale;
        for (;;) {
            // the zone (bottom, origin] is what these three say, however the bins were rounded
            origin = from > 0 ? m - from / per_bin : m;
            bottom = to < kBins - 1 ? m - (to + 1) / per_bin : -INFINITY;
            scale = per_bin * kBins / (to + 1 - from);
            __syncthreads();
            clear_bins();
            u64 total = 0, over = 0;
            int count = 0;
            row.each_with([&](float top) { return top > under; },
                          [&](const float (&v)[V], int) {
                              u64 w[V];
                              f(v, w);
#pragma unroll
                              for (int e = 0; e < V; ++e) {
                                  w[e] = v[e] > under ? w[e] : 0;
                                  total += w[e];
                                  over += v[e] > origin ? w[e] : 0;
                                  count += __popcll(__ballot(v[e] > origin));
                                  if (v[e] > fmaxf(bottom, under) && v[e] <= origin)
                                      atomicAdd(&s.bins[bin_of(v[e], origin, scale)], w[e]);
                              }
                          });
            if (t % kWave == 0) atomicAdd(&s.count, count);
            block_totals(total, over);
            over_count = s.count;
            if (t < kWave) {
                const double border = border_of(total);
                u64 before = 0;
                const int bin = static_cast<double>(over) < border ? find_bin(s.bins, over, border, before) : -1;
                if (t == 0) {
                    s.border = border;
                    s.above = before;
                    s.bin = bin;
                }
            }
            __syncthreads();
            above = s.above;
            if (s.bin >= 0) break;
            if (from == 0 && to == kBins - 1) return false;
            from = 0, to = kBins - 1;
        }
        // the keys of the bin, whether they occur or not
        unsigned low, high;
        if (t < kWave) {
            const int bin = s.bin;
            const float least_of_zone = fmaxf(bottom, under);
            const unsigned first = least_of_zone == -INFINITY ? ordered(-FLT_MAX) : ordered(least_of_zone) + 1;
            const unsigned last = ordered(fminf(origin, m));
            low = first_key(first, last, [&](unsigned k) { return bin_of(from_ordered(k), origin, scale) <= bin; });
            high = bin_of(from_ordered(last), origin, scale) >= bin
                       ? last
                       : first_key(low, last, [&](unsigned k) { return bin_of(from_ordered(k), origin, scale) < bin; }) - 1;
            if (t == 0) {
                s.low = low;
                s.high = high;
            }
        }
        __syncthreads();
        // of which the type holds only those whose last bits are clear (as a negative value's key: set)
        constexpr int kShift = T::kKeyShift;
        constexpr unsigned kRest = (1u << kShift) - 1;
        low = s.low;
        high = s.high;
        low = low >> 31 ? (low + kRest) & ~kRest : low | kRest;
        high = high >> 31 ? high & ~kRest : ((high + 1) & ~kRest) - 1;
        const float least = from_ordered(low), most = from_ordered(high);
        low >>= kShift;
        high >>= kShift;
        unsigned prefix = low;  // the keys still searched agree with it above `bits`
        int bits = low == high ? 0 : 32 - __clz(low ^ high);
        while (bits > 0) {
            const int digit = min(bits, kDigit), shift = bits - digit;
            __syncthreads();
            clear_bins();
            row.each([&](const float (&v)[V], int) {
                bool any = false;
#pragma unroll
                for (int e = 0; e < V; ++e) any |= (v[e] >= least) & (v[e] <= most);
                if (!any) return;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const unsigned k = ordered(v[e]) >> kShift;
                    if (!(v[e] >= least) || !(v[e] <= most) || (bits < 32 && ((k ^ prefix) >> bits))) continue;
                    const float one[1] = {v[e]};
                    u64 w[1];
                    f(one, w);
                    atomicAdd(&s.bins[kBins - 1 - ((k >> shift) & ((1u << digit) - 1))], w[0]);
                }
            });
            __syncthreads();
            if (t < kWave) {
                u64 before;
                const int found = find_bin(s.bins, s.above, s.border, before);
                if (t == 0) {
                    s.above = before;
                    s.bin = found;
                }
            }
            __syncthreads();
            const unsigned value = static_cast<unsigned>(kBins - 1 - s.bin) & ((1u << digit) - 1);
            const unsigned mask = bits < 32 ? (1u << bits) - 1 : 0xffffffffu;
            prefix = (prefix & ~mask) | (value << shift);
            bits = shift;
        }
        key = prefix << kShift;
        if (!(key >> 31)) key |= kRest;
        above = s.above;
        return true;
    }

    // The first k of the order by way of a short list, where k is small: the k-th largest of the threads' maxima bounds
    // the k-th largest of all from below, and few other values lie above it.  Leaves the list sorted, the order's first
    // first, and returns its length; 0 if it came out too long.
    __device__ __forceinline__ int shortlist(int k, float mine) {
        clear_bins();
        const int bin = masked(mine) ? kBins : bin_of(mine, m, per_bin);
        if (bin < kBins) atomicAdd(&s.bins[bin], 1ULL);
        __syncthreads();
        if (t < kWave) {
            u64 before;
            const int found = find_bin(s.bins, 0, static_cast<double>(k), before);
            if (t == 0) s.bin = found;
        }
        __syncthreads();
        if (s.bin < 0) return 0;  // fewer threads than k hold a value
        if (bin <= s.bin) atomicMin(&s.low, ordered(mine));
        __syncthreads();
        const float least = from_ordered(s.low);
        row.each_with(
            [&](float top) { return top >= least; },
            [&](const float (&v)[V], int first) {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    if (!(v[e] >= least)) continue;
                    const int at = atomicAdd(&s.count, 1);
                    if (at < kCandidates) s.list[at] = (static_cast<u64>(ordered(v[e])) << 32) | ~static_cast<unsigned>(first + e);
                }
            });
        __syncthreads();
        const int count = s.count;
        if (count > min(kCandidates, Group)) return 0;
        if (count <= kRanked) place(count);
        else sort(count);
        return count;
    }

    // Puts each of the list's first `count` where it belongs, by how many are larger.
    __device__ __forceinline__ void place(int count) {
        if (t == 0) s.list[count] = 0;  // the pairs below may end with it
        __syncthreads();
        u64 x = 0;
        int rank = 0;
        if (t < count) {
            x = s.list[t];
            const ulonglong2* pairs = reinterpret_cast<const ulonglong2*>(s.list);
#pragma unroll 4
            for (int i = 0; i < (count + 1) / 2; ++i) {
                const ulonglong2 pair = pairs[i];
                rank += (pair.x > x) + (pair.y > x);
            }
        }
        __syncthreads();
        if (t < count) s.list[rank] = x;
        __syncthreads();
    }

    // Descending bitonic sort of the list's first `count`, one a thread; partners within a wave exchange by shuffles.
    __device__ __forceinline__ void sort(int count) {
        int size = kWave;
        while (size < count) size *= 2;
        u64 x = t < count ? s.list[t] : 0;
        __syncthreads();
        if (t < size) {
            for (int run = 2; run <= kWave; run *= 2)
                for (int by = run / 2; by > 0; by /= 2) x = exchange(x, __shfl_xor(x, by, kWave), by, run);
        }
        for (int run = 2 * kWave; run <= size; run *= 2) {
            for (int by = run / 2; by >= kWave; by /= 2) {
                if (t < size) s.list[t] = x;
                __syncthreads();
                if (t < size) x = exchange(x, s.list[t ^ by], by, run);
                __syncthreads();
            }
            if (t < size)
                for (int by = kWave / 2; by > 0; by /= 2) x = exchange(x, __shfl_xor(x, by, kWave), by, run);
        }
        if (t < size) s.list[t] = x;
        __syncthreads();
    }
    __device__ __forceinline__ u64 exchange(u64 x, u64 other, int by, int run) const {
        const bool larger = ((t & run) == 0) == ((t & by) == 0);
        return (x > other) == larger ? x : other;
    }

    // Inclusive prefix sum over the workgroup's threads.
    __device__ __forceinline__ u64 scan(u64 v) {
        v = wave_scan(v);
        if (t % kWave == kWave - 1) s.sums[t / kWave] = v;
        __syncthreads();
        for (int i = 0; i < t / kWave; ++i) v += s.sums[i];
        return v;
    }
};

template <typename T, int Group, bool Held, int Segments>
__global__ __launch_bounds__(Group) void sample_block(Params p) {
    typedef typename T::Store Store;
    typedef Team<Group> G;
    constexpr int V = T::kPerChunk;
    __shared__ Shared s;
    __shared__ u64 mass[Segments];
    __shared__ int tied[Segments];
    const long long r = blockIdx.x;
    const int t = static_cast<int>(threadIdx.x), lane = t % kWave;
    tokens::LongRow<T, Group, Held> row;
    row.open(static_cast<const Store*>(p.logits) + r * p.ld, p.classes);
    fill_table(s.table);  // under the row's loads
    const Settings set(p, r);
    float mine = -INFINITY;
    row.each_max([&](float top) { mine = fmaxf(mine, top); });
    const float m = G::max(mine, s.reduce);
    if (!set.valid || m == -INFINITY) {
        if (t == 0) nothing_drawn(p, r, set.valid);
        return;
    }
    const Weights weight(s.table, m, set.per_t);
    Sampler<T, Group, Held> sampler{row, s, t, m, static_cast<float>(kBinsPerUnit * set.per_t)};

    // what stays of the order: keys above `key`, and the first `ties` (by index) of those equal to it
    unsigned key = 0;
    int ties = INT_MAX;
    if (set.one()) {
        key = ordered(m);
        ties = 1;
    } else {
        unsigned cut;
        u64 above;
        const bool top_k = set.top_k > 0 && set.top_k < p.classes;
        const int listed = top_k && set.top_k <= Group / 2 ? sampler.shortlist(set.top_k, mine) : 0;
        if (listed) {
            // the list holds the order's first `listed`: weights and borders from there
            const u64 entry = t < listed ? s.list[t] : 0;
            const unsigned own = static_cast<unsigned>(entry >> 32);
            u64 w = t < min(set.top_k, listed) ? weight(from_ordered(own)) : 0;
            const u64 upto = sampler.scan(w);
            __syncthreads();
            if (t == Group - 1) s.above = upto;
            if (t == 0) s.count = 0;
            __syncthreads();
            const double border = set.top_p < 1.0 ? set.top_p * static_cast<double>(s.above) : INFINITY;
            const bool stays = t < min(set.top_k, listed) &&
                               (t == 0 || (static_cast<double>(upto - w) < border && w >= set.min_weight));
            const u64 votes = __ballot(stays);
            if (lane == 0 && votes) atomicAdd(&s.count, __popcll(votes));
            __syncthreads();
            const int kept = s.count;
            if (kept <= kWave) {
                // wave 0 has them all: the running sums by index
                if (t >= kWave) return;
                w = t < kept ? w : 0;
                const unsigned index = ~static_cast<unsigned>(entry);
                u64 run = 0, total = 0;
                for (int i = 0; i < kept; ++i) {
                    const u64 other = lane64(w, i);
                    total += other;
                    run += static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(index), i)) <= index ? other : 0;
                }
                const double target = set.target(total);
                // of those whose running sum passes the target the one of the lowest index
                const unsigned first = wave_min(t < kept && static_cast<double>(run) > target ? index : 0xffffffffu);
                if (t < kept && index == first) drawn(p, r, index, from_ordered(own), m, set.per_t, total);
                return;
            }
            __syncthreads();
            if (t == kept - 1) s.low = own;
            if (t == 0) s.count = 0;
            __syncthreads();
            key = s.low;
            const u64 equal = __ballot(t < kept && own == key);
            if (lane == 0 && equal) atomicAdd(&s.count, __popcll(equal));
            __syncthreads();
            ties = s.count;
        } else {
            if (top_k) __syncthreads();
            if (top_k && sampler.cut_at(Ones(), CountBorder{set.top_k}, 0u, mine, cut, above)) {
                key = cut;
                ties = set.top_k - static_cast<int>(above);
            }
            if (set.top_p < 1.0) {
                __syncthreads();
                const bool limited = ties != INT_MAX;
                u64 tie = limited ? weight(from_ordered(key)) : 0;
                const ShareBorder border{set.top_p, limited ? tie * static_cast<u64>(ties) : 0};
                const bool found = sampler.cut_at(weight, border, limited ? key : 0u, mine, cut, above);
                if (found) {
                    key = cut;
                    tie = weight(from_ordered(key));
                    ties = p.classes;
                }
                if ((found || limited) && tie > 0) ties = ties_below(s.border, above, tie, ties);
            }
        }
    }
    const float least = key ? from_ordered(key) : -FLT_MAX;
    u64 tie = ties == INT_MAX ? 0 : weight(least);
    if (tie < set.min_weight) tie = 0;

    // kept mass (without ties) and ties of every segment of 64 chunks, in index order
    const bool cuts = ties != INT_MAX;
    const auto kept = [&](const float (&v)[V], u64 (&w)[V]) {
        weight(v, w);
#pragma unroll
        for (int e = 0; e < V; ++e) w[e] = w[e] < set.min_weight || (cuts && !(v[e] > least)) ? 0 : w[e];
    };
    const int segments = row.passes() * G::kWaves;
    // no value below can stay: the border, and min-p's with room for its rounding
    const float lowest = fmaxf(least, set.min_weight ? __double2float_rd(m + (log(set.min_weight / kScale) - 1e-3) / set.per_t)
                                                     : -FLT_MAX);
    bool summed = false;
    if ((cuts || set.min_weight) && sampler.over_count <= kKept && lowest > -FLT_MAX && lowest < INFINITY) {
        // where few values stay they are listed first, and only these weighed; if most threads hold one there are many
        __syncthreads();
        for (int g = t; g < segments; g += Group) mass[g] = 0, tied[g] = 0;
        if (t == 0) s.count = 0, s.high = 0;
        __syncthreads();
        const u64 holders = __ballot(mine >= lowest);
        if (lane == 0) atomicAdd(&s.high, static_cast<unsigned>(__popcll(holders)));
        __syncthreads();
        int count = kKept + 1;
        if (s.high * 8 <= Group * 7) {
            row.each_pass([&](int i, const float (&v)[V], float top) {
                if (!(top >= lowest)) return;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    if (!(v[e] >= lowest)) continue;
                    const int at = atomicAdd(&s.count, 1);
                    if (at < kKept) {
                        s.kept[at].value = v[e];
                        s.kept[at].segment = i * G::kWaves + t / kWave;
                    }
                }
            });
            __syncthreads();
            count = s.count;
        }
        summed = count <= kKept;
        if (summed) {
            for (int at = t; at < count; at += Group) {
                const float z = s.kept[at].value;
                const int g = s.kept[at].segment;
                const u64 w = weight(z);
                if (cuts && z == least) atomicAdd(&tied[g], 1);
                else if (w >= set.min_weight) atomicAdd(&mass[g], w);
            }
        }
    }
    if (!summed) {
        __syncthreads();
        row.each_pass([&](int i, const float (&v)[V], float top) {
            u64 sum = 0;
            int equal = 0;
            if (__ballot(top >= lowest)) {
                u64 w[V];
                kept(v, w);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    sum += w[e];
                    equal += cuts && v[e] == least;
                }
                sum = wave_total(sum);
                if (cuts) equal = wave_total(equal);
            }
            if (lane == 0) {
                mass[i * G::kWaves + G::wave()] = sum;
                tied[i * G::kWaves + G::wave()] = equal;
            }
        });
    }
    __syncthreads();
    if (t >= kWave) return;

    // wave 0: the ties that stay in each segment, the sum of all, and the segment where it passes u
    u64 total = 0;
    int ties_before = 0;
    for (int first = 0; first < segments; first += kWave) {
        const int g = first + lane;
        const int equal = g < segments ? tied[g] : 0;
        const int upto = ties_before + wave_scan(equal);
        const int before = upto - equal;
        u64 sum = 0;
        if (g < segments) {
            sum = mass[g] + static_cast<u64>(max(min(ties - before, equal), 0)) * tie;
            mass[g] = sum;
            tied[g] = before;
        }
        total += wave_total(sum);
        ties_before = __builtin_amdgcn_readlane(upto, kWave - 1);
    }
    Team<kWave>::sync();
    const double target = set.target(total);
    u64 before = 0;
    int segment = -1;
    for (int first = 0; first < segments && segment < 0; first += kWave) {
        const int g = first + lane;
        const u64 sum = g < segments ? mass[g] : 0;
        const u64 upto = before + wave_scan(sum);
        const u64 found = __ballot(static_cast<double>(upto) > target);
        if (found) {
            const int at = __ffsll(found) - 1;
            segment = first + at;
            before = lane64(upto - sum, at);
        } else {
            before = lane64(upto, kWave - 1);
        }
    }

    // the segment's chunks, one a lane
    float v[V];
    const int chunk = segment * kWave + lane;
    T::unpack(row.read(chunk), v);
    int equal = 0;
#pragma unroll
    for (int e = 0; e < V; ++e) equal += cuts && v[e] == least;
    int rank = tied[segment] + wave_scan(equal) - equal;
    u64 w[V], sum = 0;
    kept(v, w);
#pragma unroll
    for (int e = 0; e < V; ++e) {
        if (cuts && v[e] == least) w[e] = rank++ < ties ? tie : 0;
        sum += w[e];
    }
    const u64 upto = before + wave_scan(sum);
    const u64 found = __ballot(static_cast<double>(upto) > target);
    if (lane != __ffsll(found) - 1) return;
    u64 run = upto - sum;
    int at = -1;
    float chosen = m;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        run += w[e];
        if (at < 0 && static_cast<double>(run) > target) {
            at = chunk * V + e;
            chosen = v[e];
        }
    }
    drawn(p, r, at, chosen, m, set.per_t, total);
}

template <typename T, int Lanes, int E>
void launch_short(const Params& p, hipStream_t stream) {
    hipLaunchKernelGGL((sample_short<T, Lanes, E>), tokens::grid_for(p.rows, kShortThreads / Lanes, kShortThreads),
                       dim3(kShortThreads), 0, stream, p);
}

template <typename T, int Group, bool Held>
void launch_block(const Params& p, hipStream_t stream) {
    constexpr int kSegments = Held ? tokens::kHeldChunks * Group / kWave : kMaxClasses / (kWave * T::kPerChunk);
    hipLaunchKernelGGL((sample_block<T, Group, Held, kSegments>), tokens::grid_for(p.rows, 1, Group), dim3(Group), 0, stream, p);
}

template <typename T>
void launch(const Params& p, hipStream_t stream) {
    constexpr int kHeld = tokens::kHeldChunks * T::kPerChunk;  // classes a thread can hold
    if (p.classes <= 32) launch_short<T, 16, 2>(p, stream);
    else if (p.classes <= 64) launch_short<T, 16, 4>(p, stream);
    else if (p.classes <= 128) launch_short<T, 16, 8>(p, stream);
    else if (p.classes <= 256) launch_short<T, 16, 16>(p, stream);
    else if (p.classes <= 512) launch_short<T, 64, 8>(p, stream);
    else if (p.classes <= 1024) launch_short<T, 64, 16>(p, stream);
    else if (p.classes <= 256 * kHeld && (p.rows > 512 || p.classes <= 4096)) launch_block<T, 256, true>(p, stream);
    else if (p.classes <= 1024 * kHeld) launch_block<T, 1024, true>(p, stream);
    else launch_block<T, 1024, false>(p, stream);
}

}  // namespace sample
}  // namespace rl

RL_API int rl_categorical_sample(const void* logits, int type, long long ld, long long rows, int classes,
                                 double temperature, int top_k, double top_p, double min_p,
                                 const float* temperature_rows, const int* top_k_rows, const float* top_p_rows,
                                 const float* min_p_rows, const float* uniform, long long* tokens_out, float* log_probs,
                                 void* stream) {
    return rl::guarded("rl_categorical_sample", [&] {
        using namespace rl;
        require(tokens::known_type(type), "Sampling takes logits of type 0 (fp32), 1 (bf16) or 3 (fp16).");
        require(rows >= 0 && classes > 0 && classes <= sample::kMaxClasses,
                "Sampling takes no negative number of rows and 1 to 2^20 classes.");
        require(rows == 0 || (logits && uniform && tokens_out), "Sampling operands must be nonnull.");
        require(rows <= 1 || ld >= classes, "The rows of logits overlap.");
        require(aligned(logits, tokens::type_size(type)), "The logits must be aligned to their elements.");
        require(temperature_rows || (temperature >= 0.0 && std::isfinite(temperature)),
                "The temperature must be finite and not negative.");
        require(top_p_rows || !std::isnan(top_p), "top_p is not a number.");
        require(min_p_rows || !std::isnan(min_p), "min_p is not a number.");
        if (rows == 0) return;
        sample::Params p{logits, ld, rows, classes, temperature, top_p, min_p, top_k, temperature_rows, top_p_rows,
                         min_p_rows, top_k_rows, uniform, tokens_out, log_probs};
        if (type == tokens::kF32) sample::launch<tokens::F32>(p, as_stream(stream));
        else if (type == tokens::kBf16) sample::launch<tokens::Bf16>(p, as_stream(stream));
        else sample::launch<tokens::F16>(p, as_stream(stream));
        check_launch("Launch sampling");
    });
}
