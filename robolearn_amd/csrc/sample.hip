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
// rounded once to a multiple of 2^-43 (2^-44 off at most; 2^20 classes of weight 1 sum to 2^63).  Integer sums have no
// order: histograms by LDS atomics and sums over waves in any order give the same token on every run.
//
// One group of threads a row.  No sort: a cut (top-k by counts, top-p by mass) is found from a histogram over the
// distance to the maximum, 1024 bins of which the border lies in one, and then by digits of the order-preserving bits
// of the logits in that bin.  The result is a border key, how many tokens of exactly that key stay (by index), and the
// mass above.  The last pass sums the kept weights of 64-chunk segments in index order; the segment that holds the
// token is scanned by one wave.
#include "tokens.hpp"

#include <climits>
#include <cmath>

namespace rl {
namespace sample {

using tokens::Row;
using tokens::Team;

typedef unsigned long long u64;

constexpr int kMaxClasses = 1 << 20;
constexpr int kBins = 1024;
constexpr int kBinsPerLane = kBins / kWave;
constexpr int kDigit = 10;             // bits of a digit: a bin each
static_assert(kBins == 1 << kDigit, "a bin for each digit");
constexpr float kBinsPerUnit = 32.0f;  // linear bins of 1/32 of (max - z) / T: 32 units until the last one

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

// Bits that order as the values do (NaN excluded, -0 as 0).
__device__ __forceinline__ unsigned ordered(float z) {
    const unsigned b = __float_as_uint(z + 0.0f);
    return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ bool masked(float z) { return !(z > -INFINITY); }  // -infinity or NaN

// exp((z - m) / T) in 64 bits; m itself weighs 1 whatever it is.
__device__ __forceinline__ double weight(float z, float m, double per_t) {
    if (z == m) return 1.0;
    if (masked(z)) return 0.0;
    return exp((static_cast<double>(z) - static_cast<double>(m)) * per_t);
}

// A weight of [0, 1] as a multiple of 2^-43, rounded to nearest: the sum with 2^9 holds 2^-43 in its last bit.
__device__ __forceinline__ u64 fixed(double w) {
    return static_cast<u64>(__double_as_longlong(w + 512.0) - __double_as_longlong(512.0));
}

__device__ __forceinline__ u64 shuffle_up(u64 v, int by) { return __shfl_up(v, by, kWave); }

// Inclusive prefix sum over a wave.
__device__ __forceinline__ u64 wave_scan(u64 v) {
    const int lane = threadIdx.x % kWave;
#pragma unroll
    for (int by = 1; by < kWave; by *= 2) {
        const u64 o = shuffle_up(v, by);
        if (lane >= by) v += o;
    }
    return v;
}

__device__ __forceinline__ u64 wave_total(u64 v) {
#pragma unroll
    for (int by = 32; by > 0; by /= 2) v += __shfl_xor(v, by, kWave);
    return v;
}

template <int Group>
struct Shared {
    u64 bins[kBins];
    u64 above;      // running sum before the bin found
    double border;
    int bin;
    unsigned low, high;
    float reduce[Team<Group>::kWaves];
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
        before = __shfl(upto, kWave - 1, kWave);
        return -1;
    }
    const int first = __ffsll(found) - 1;
    u64 sum = __shfl(upto - mine, first, kWave);
    int bin = first * kBinsPerLane;
    for (int i = 0; i < kBinsPerLane; ++i, ++bin) {
        const u64 next = sum + bins[first * kBinsPerLane + i];
        if (static_cast<double>(next) >= border) break;
        sum = next;
    }
    before = sum;
    return bin;
}

template <typename T, int Group, int Held>
struct Sampler {
    typedef Team<Group> G;
    typedef Row<T, Group, Held> R;
    static constexpr int V = T::kPerChunk;

    const R& row;
    Shared<Group>& s;
    const int t;
    const float m;         // the row's maximum
    const double per_t;
    const float per_bin;   // bins of a unit of logits

    __device__ __forceinline__ int bin_of(float z) const {
        if (z == m) return 0;
        const float d = (m - z) * per_bin;
        return d < kBins - 1 ? static_cast<int>(d) : kBins - 1;
    }

    __device__ __forceinline__ void clear_bins() {
        for (int b = t; b < kBins; b += Group) s.bins[b] = 0;
        if (t == 0) {
            s.low = 0xffffffffu;
            s.high = 0;
        }
        G::sync();
    }

    // The key, above `floor`, at which the running sum of f reaches border_of(sum of all): in `key`, with the sum of
    // the keys above it in `above`.  False if none does; `above` is then the sum of all.  The border must be positive.
    template <typename F, typename B>
    __device__ __forceinline__ bool cut_at(F f, B border_of, unsigned floor, unsigned& key, u64& above) {
        clear_bins();
        row.each([&](int, const float (&v)[V], int) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                if (masked(v[e]) || ordered(v[e]) <= floor) continue;
                atomicAdd(&s.bins[bin_of(v[e])], f(v[e]));
            }
        });
        G::sync();
        if (t < kWave) {
            u64 all = 0;
#pragma unroll
            for (int i = 0; i < kBinsPerLane; ++i) all += s.bins[t * kBinsPerLane + i];
            const double border = border_of(wave_total(all));
            u64 before;
            const int bin = find_bin(s.bins, 0, border, before);
            if (t == 0) {
                s.border = border;
                s.above = before;
                s.bin = bin;
            }
        }
        G::sync();
        const int bin = s.bin;
        above = s.above;
        if (bin < 0) return false;
        // the bin's keys: digits from the first bit in which they differ
        unsigned low = 0xffffffffu, high = 0;
        row.each([&](int, const float (&v)[V], int) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const unsigned k = ordered(v[e]);
                if (masked(v[e]) || k <= floor || bin_of(v[e]) != bin) continue;
                low = min(low, k);
                high = max(high, k);
            }
        });
        if (low <= high) {
            atomicMin(&s.low, low);
            atomicMax(&s.high, high);
        }
        G::sync();
        low = s.low;
        high = s.high;
        unsigned prefix = low;  // the keys still searched agree with it above `bits`
        int bits = low == high ? 0 : 32 - __clz(low ^ high);
        while (bits > 0) {
            const int digit = min(bits, kDigit), shift = bits - digit;
            G::sync();
            clear_bins();
            row.each([&](int, const float (&v)[V], int) {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const unsigned k = ordered(v[e]);
                    if (masked(v[e]) || k <= floor || bin_of(v[e]) != bin) continue;
                    if (bits < 32 && ((k ^ prefix) >> bits)) continue;
                    atomicAdd(&s.bins[kBins - 1 - ((k >> shift) & ((1u << digit) - 1))], f(v[e]));
                }
            });
            G::sync();
            if (t < kWave) {
                u64 before;
                const int found = find_bin(s.bins, s.above, s.border, before);
                if (t == 0) {
                    s.above = before;
                    s.bin = found;
                }
            }
            G::sync();
            const unsigned value = static_cast<unsigned>(kBins - 1 - s.bin) & ((1u << digit) - 1);
            const unsigned mask = bits < 32 ? (1u << bits) - 1 : 0xffffffffu;
            prefix = (prefix & ~mask) | (value << shift);
            bits = shift;
        }
        key = prefix;
        above = s.above;
        return true;
    }
};

// The logit whose ordered bits are `key`.
__device__ __forceinline__ float from_ordered(unsigned key) {
    return __uint_as_float(key ^ (key >> 31 ? 0x80000000u : 0xffffffffu));
}

template <typename T, int Group, int Held, int Segments>
__global__ __launch_bounds__(Group < 256 ? 256 : Group) void sample_kernel(Params p) {
    typedef typename T::Store Store;
    typedef Team<Group> G;
    constexpr int kTeams = Group < 256 ? 256 / Group : 1;
    constexpr int V = T::kPerChunk;
    __shared__ Shared<Group> shared[kTeams];
    __shared__ u64 segment_mass[kTeams][Segments];
    __shared__ int segment_ties[kTeams][Segments];
    const int team = static_cast<int>(threadIdx.x) / Group % kTeams;
    Shared<Group>& s = shared[team];
    u64* mass = segment_mass[team];
    int* tied = segment_ties[team];

    const long long r = blockIdx.x * static_cast<long long>(kTeams) + threadIdx.x / Group;
    if (r >= p.rows) return;  // a team of its own wave, or none of the workgroup
    const int t = G::thread(), lane = t % kWave;
    const double temperature = p.temperatures ? p.temperatures[r] : p.temperature;
    const double top_p = p.top_ps ? p.top_ps[r] : p.top_p;
    const double min_p = fmin(p.min_ps ? p.min_ps[r] : p.min_p, 1.0);
    const int top_k = p.top_ks ? p.top_ks[r] : p.top_k;
    const float u = p.uniform[r];
    const bool valid = temperature >= 0.0 && temperature < INFINITY && top_p == top_p &&
                       (p.min_ps ? p.min_ps[r] == p.min_ps[r] : true) && u == u;

    Row<T, Group, Held> row;
    row.open(static_cast<const Store*>(p.logits) + r * p.ld, p.classes);
    float m = -INFINITY;
    row.each([&](int, const float (&v)[V], int) {
#pragma unroll
        for (int e = 0; e < V; ++e) m = fmaxf(m, v[e]);
    });
    m = G::max(m, s.reduce);
    if (!valid || m == -INFINITY) {
        if (t == 0) {
            p.tokens[r] = -1;
            if (p.log_probs) p.log_probs[r] = valid ? -INFINITY : NAN;
        }
        return;
    }
    const bool greedy = temperature == 0.0;
    const double per_t = greedy ? 0.0 : 1.0 / temperature;
    const float per_bin = static_cast<float>(kBinsPerUnit * per_t);
    Sampler<T, Group, Held> sampler{row, s, t, m, per_t, per_bin};

    // what stays of the order: keys above `key`, and the first `ties` (by index) of those equal to it
    unsigned key = 0;
    int ties = INT_MAX;
    if (greedy || top_p <= 0.0 || top_k == 1) {
        key = ordered(m);
        ties = 1;
    } else {
        unsigned cut;
        u64 above;
        if (top_k > 0 && top_k < p.classes &&
            sampler.cut_at([](float) { return 1ULL; }, [&](u64) { return static_cast<double>(top_k); }, 0u, cut, above)) {
            key = cut;
            ties = top_k - static_cast<int>(above);
        }
        if (top_p < 1.0) {
            G::sync();
            const bool limited = ties != INT_MAX;
            u64 tie = limited ? fixed(weight(from_ordered(key), m, per_t)) : 0;
            const u64 tied = limited ? tie * static_cast<u64>(ties) : 0;
            const bool found = sampler.cut_at([&](float z) { return fixed(weight(z, m, per_t)); },
                                              [&](u64 all) { return top_p * static_cast<double>(all + tied); },
                                              limited ? key : 0u, cut, above);
            if (found) {
                key = cut;
                tie = fixed(weight(from_ordered(key), m, per_t));
                ties = p.classes;
            }
            // the i-th of the equal keys stays while the mass before it, above + i tie, is below the border
            if ((found || limited) && tie > 0) {
                const double stay = ceil((s.border - static_cast<double>(above)) / static_cast<double>(tie));
                ties = static_cast<int>(fmax(fmin(stay, static_cast<double>(ties)), 1.0));
            }
        }
    }
    const double tie_weight = ties == INT_MAX ? 0.0 : weight(from_ordered(key), m, per_t);
    const u64 tie = tie_weight >= min_p ? fixed(tie_weight) : 0;

    // kept mass (without ties) and ties of every segment of 64 chunks, in index order
    const auto kept = [&](float z) -> u64 {
        if (masked(z) || ordered(z) <= key) return 0;
        const double w = weight(z, m, per_t);
        return w >= min_p ? fixed(w) : 0;
    };
    const auto is_tie = [&](float z) { return !masked(z) && ordered(z) == key; };
    const int segments = row.passes() * G::kWaves;
    row.each([&](int i, const float (&v)[V], int) {
        if (i >= row.passes()) return;
        u64 sum = 0;
        int equal = 0;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            sum += kept(v[e]);
            equal += is_tie(v[e]);
        }
        sum = wave_total(sum);
        equal = static_cast<int>(wave_total(static_cast<u64>(equal)));
        if (lane == 0) {
            mass[i * G::kWaves + G::wave()] = sum;
            tied[i * G::kWaves + G::wave()] = equal;
        }
    });
    G::sync();
    if (t >= kWave) return;

    // wave 0: the ties that stay in each segment, the sum of all, and the segment where it passes u
    u64 total = 0;
    int ties_before = 0;
    for (int first = 0; first < segments; first += kWave) {
        const int g = first + lane;
        const int equal = g < segments ? tied[g] : 0;
        const int upto = ties_before + static_cast<int>(wave_scan(static_cast<u64>(equal)));
        const int before = upto - equal;
        u64 sum = 0;
        if (g < segments) {
            sum = mass[g] + static_cast<u64>(max(min(ties - before, equal), 0)) * tie;
            mass[g] = sum;
            tied[g] = before;
        }
        total += wave_total(sum);
        ties_before = __shfl(upto, kWave - 1, kWave);
    }
    Team<kWave>::sync();
    const double target = fmax(fmin(static_cast<double>(u), 1.0 - 0x1p-50), 0.0) * static_cast<double>(total);
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
            before = __shfl(upto - sum, at, kWave);
        } else {
            before = __shfl(upto, kWave - 1, kWave);
        }
    }

    // the segment's chunks, one a lane
    float v[V];
    const int chunk = segment * kWave + lane;
    T::unpack(row.read(chunk), v);
    int equal = 0;
#pragma unroll
    for (int e = 0; e < V; ++e) equal += is_tie(v[e]);
    int rank = tied[segment] + static_cast<int>(wave_scan(static_cast<u64>(equal))) - equal;
    u64 w[V], sum = 0;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        w[e] = is_tie(v[e]) ? (rank++ < ties ? tie : 0) : kept(v[e]);
        sum += w[e];
    }
    const u64 upto = before + wave_scan(sum);
    const u64 found = __ballot(static_cast<double>(upto) > target);
    if (lane != __ffsll(found) - 1) return;
    u64 run = upto - sum;
    bool done = false;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        run += w[e];
        if (done || !(static_cast<double>(run) > target)) continue;
        done = true;
        p.tokens[r] = static_cast<long long>(chunk) * V + e;
        if (p.log_probs) {
            const double x = v[e] == m ? 0.0 : (static_cast<double>(v[e]) - static_cast<double>(m)) * per_t;
            p.log_probs[r] = static_cast<float>(x - log(static_cast<double>(total) * 0x1p-43));
        }
    }
}

template <typename T>
void launch(const Params& p, hipStream_t stream) {
    if (p.classes <= 64 * T::kPerChunk)
        hipLaunchKernelGGL((sample_kernel<T, 64, 1, 1>), dim3(ceil_div(p.rows, 4)), dim3(256), 0, stream, p);
    else
        hipLaunchKernelGGL((sample_kernel<T, 256, 0, kMaxClasses / (64 * T::kPerChunk)>),
                           dim3(static_cast<unsigned>(p.rows)), dim3(256), 0, stream, p);
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
        require(rows >= 0 && rows <= INT_MAX && classes > 0 && classes <= sample::kMaxClasses,
                "Sampling takes 0 to 2^31 - 1 rows of 1 to 2^20 classes.");
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
