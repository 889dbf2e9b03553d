// Distillation from a teacher's top logits: the loss of a student's row of logits and its gradient.
//
//   p = softmax(t / T) over the row's entries (t_k, i_k), q = softmax(z / T) over all classes,
//   L = w T^2 sum_k p_k (log p_k - log q[i_k]),  dL/dz_j = w T (q_j - sum_{k: i_k = j} p_k).
//
// An entry whose index lies outside [0, classes) is padding; a row without entries (or whose entries are all -infinity)
// and a row of weight 0 have loss 0 and gradient 0 whatever their logits hold.
//
// Bound by HBM where rows are long: 4096 x 32768 bf16 with 64 entries 118 us for loss and gradient (4.6 TB/s of logits and
// gradient, a copy of the same bytes 98 us), the gradient alone of 1000 x 50021 fp32 94 us (4.3 TB/s); what is left are
// the entries' scattered reads and writes (112 us with one entry).  Short rows are bound by their chain of loads and
// reductions: 2048 x 101 fp32 6 us, under the host's 8.
//
// One group of threads a row, the entries in LDS.  Exponents are taken of (z - max z) / T, so that their rounding is
// relative to the distance from the row's maximum, where the weight lies; sums are fp32 per thread and in a fixed
// order, the few terms of the loss in 64 bits.  The gradient is written for all classes first; then, behind a barrier,
// every entry writes its class again with all entries of that class subtracted, so that classes named twice come
// out right and no order of writes matters.
#include "tokens.hpp"

#include <cfloat>
#include <climits>
#include <cmath>

namespace rl {
namespace distill {

using tokens::Row;
using tokens::Team;

constexpr int kMaxEntries = 1024;
constexpr float kLog2e = 1.44269504088896340736f;

struct Params {
    const void* logits;
    long long ld;
    const void* teacher;     // [rows, entries], of teacher_type
    const void* index;       // [rows, entries], int64 or int32
    const float* weights;    // [rows] or null
    const float* lse_in;     // backward: logsumexp(z / T) a row
    const float* dloss;      // backward: gradient of each row's loss
    float* loss;             // forward: [rows]
    float* lse_out;          // forward: [rows] or null
    void* dlogits;           // as the logits, or null
    long long ldd;
    float grad_scale;        // forward: factor of the gradient
    double temperature, per_t;  // T, 1 / T
    float rate;                 // log2(e) / T
    long long rows;
    int classes, entries, teacher_type, index_wide;
};

__device__ __forceinline__ float teacher_value(const Params& p, long long at) {
    if (p.teacher_type == tokens::kF32) return static_cast<const float*>(p.teacher)[at];
    const unsigned short bits = static_cast<const unsigned short*>(p.teacher)[at];
    return p.teacher_type == tokens::kBf16 ? tokens::Bf16::value(bits) : tokens::F16::value(bits);
}

// LDS of a team: for every entry its logit of the teacher, its weight exp((t - max t) / T), its class and the student's
// logit there; entries up to the next multiple of 4 are padding.
struct Entries {
    float *teacher, *share, *logit;
    int* cls;
    int padded;

    __host__ __device__ static int round4(int entries) { return (entries + 3) / 4 * 4; }
    __device__ __forceinline__ Entries(unsigned char* lds, int team, int entries) : padded(round4(entries)) {
        teacher = reinterpret_cast<float*>(lds) + team * 4 * padded;
        share = teacher + padded;
        logit = share + padded;
        cls = reinterpret_cast<int*>(logit + padded);
    }
    // the weights of all entries of class c
    __device__ __forceinline__ float share_of(int c) const {
        float sum = 0.0f;
#pragma unroll 4
        for (int o = 0; o < padded; o += 4) {
            const int4 k = *reinterpret_cast<const int4*>(cls + o);
            const float4 e = *reinterpret_cast<const float4*>(share + o);
            sum += k.x == c ? e.x : 0.0f;
            sum += k.y == c ? e.y : 0.0f;
            sum += k.z == c ? e.z : 0.0f;
            sum += k.w == c ? e.w : 0.0f;
        }
        return sum;
    }
};

template <typename T, int Group, int Held, bool Backward>
__global__ __launch_bounds__(Group < 256 ? 256 : Group) void distill_kernel(Params p) {
    typedef typename T::Store Store;
    typedef Team<Group> G;
    constexpr int kTeams = Group < 256 ? 256 / Group : 1;
    constexpr int V = T::kPerChunk;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    __shared__ float scratch_all[kTeams][2 * G::kWaves];
    const int team = static_cast<int>(threadIdx.x) / Group % kTeams;
    float* scratch = scratch_all[team];
    const Entries entry(lds, team, p.entries);

    const long long row = blockIdx.x * static_cast<long long>(kTeams) + team;
    if (row >= p.rows) return;  // a team inside a wave, or none of the workgroup
    const int t = G::thread();
    const Store* z = static_cast<const Store*>(p.logits) + row * p.ld;
    Store* dz = p.dlogits ? static_cast<Store*>(p.dlogits) + row * p.ldd : nullptr;
    Row<T, Group, Held> r;
    r.open(z, p.classes);
    const float weight = p.weights ? p.weights[row] : 1.0f;
    const float rate = p.rate;

    // the entries, and both maxima
    float top[2] = {-INFINITY, -INFINITY};  // the teacher's, the student's
    bool bad = false;                       // a NaN among the entries
    for (int k = t; k < entry.padded; k += Group) {
        const long long at = row * p.entries + k;
        const bool real = k < p.entries;
        const long long c = !real ? -1
                            : p.index_wide ? static_cast<const long long*>(p.index)[at]
                                           : static_cast<long long>(static_cast<const int*>(p.index)[at]);
        const bool valid = c >= 0 && c < p.classes;
        const float x = valid ? teacher_value(p, at) : -INFINITY;
        entry.teacher[k] = x;
        entry.cls[k] = valid ? static_cast<int>(c) : -1;
        entry.logit[k] = valid ? T::value(z[c]) : -INFINITY;
        top[0] = fmaxf(top[0], x);
        bad |= x != x;
    }
    if (bad) top[0] = INFINITY;  // infinity - infinity below: the row's loss is NaN
    float sums[2] = {0.0f, 1.0f};
    if constexpr (!Backward) {
        if constexpr (Held > 0) {
            r.each([&](int, const float (&v)[V], int) {
#pragma unroll
                for (int e = 0; e < V; ++e) top[1] = fmaxf(top[1], v[e]);
            });
        } else {
            // one pass: a running maximum, and the sum relative to it
            float s = 0.0f;
            r.each([&](int, const float (&v)[V], int) {
                float high = top[1];
#pragma unroll
                for (int e = 0; e < V; ++e) high = fmaxf(high, v[e]);
                if (high == -INFINITY) return;
                s *= __builtin_amdgcn_exp2f((top[1] - high) * rate);
#pragma unroll
                for (int e = 0; e < V; ++e) s += __builtin_amdgcn_exp2f((v[e] - high) * rate);
                top[1] = high;
            });
            sums[1] = s;
        }
    }
    const float mine = top[1];
    G::max(top, scratch);
    const float m = top[1];

    const bool empty = weight == 0.0f || top[0] == -INFINITY;
    if (empty && !(Backward ? false : p.lse_out != nullptr)) {
        if (!Backward && t == 0) p.loss[row] = 0.0f;
        if (dz) {
            G::sync();
            for (int j = t; j < p.classes; j += Group) dz[j] = Store(0);
        }
        return;
    }

    // the weights of the entries and of the classes
    for (int k = t; k < entry.padded; k += Group) {
        const float e = empty ? 0.0f : __builtin_amdgcn_exp2f((entry.teacher[k] - top[0]) * rate);
        entry.share[k] = e;
        sums[0] += e;
    }
    r.packed();
    double log_sum = 0.0;
    if constexpr (!Backward) {
        if constexpr (Held > 0) {
            sums[1] = 0.0f;
            r.each([&](int, const float (&v)[V], int) {
#pragma unroll
                for (int e = 0; e < V; ++e) sums[1] += __builtin_amdgcn_exp2f((v[e] - m) * rate);
            });
        } else if (mine != -INFINITY) {
            sums[1] *= __builtin_amdgcn_exp2f((mine - m) * rate);
        }
        G::sum(sums, scratch);
        log_sum = log(static_cast<double>(sums[1]));
        if (t == 0 && p.lse_out) p.lse_out[row] = static_cast<float>(m * p.per_t + log_sum);
        if (empty) {
            if (t == 0) p.loss[row] = 0.0f;
            if (dz) {
                G::sync();
                for (int j = t; j < p.classes; j += Group) dz[j] = Store(0);
            }
            return;
        }
    } else {
        sums[0] = G::sum(sums[0], scratch);
    }
    if (dz) {
        const float factor = static_cast<float>(weight * p.temperature * (Backward ? p.dloss[row] : p.grad_scale));
        // q(z): forward exp2((z - m) rate) / s; backward exp(z / T - lse), with 1 / T in two pieces so that the
        // difference is rounded once
        const float inverse = 1.0f / sums[1];
        const float by = static_cast<float>(p.per_t);
        const float by_rest = static_cast<float>(p.per_t - by);
        const float lse = Backward ? p.lse_in[row] : 0.0f;
        const auto q = [&](float x) {
            if constexpr (Backward) {
                x = fmaxf(x, -FLT_MAX);  // -infinity times a negative rest would be infinity
                return __builtin_amdgcn_exp2f((__builtin_fmaf(x, by, -lse) + x * by_rest) * kLog2e);
            } else {
                return __builtin_amdgcn_exp2f((x - m) * rate) * inverse;
            }
        };
        G::sync();  // every logit of the entries is read: the gradient may take the logits' place
        r.packed();
        r.each([&](int, const float (&v)[V], int first) {
            if (first >= p.classes) return;
            float d[V];
#pragma unroll
            for (int e = 0; e < V; ++e) d[e] = factor * q(v[e]);
            if (first + V <= p.classes) {
                const uint4 c = T::pack(d);
                *reinterpret_cast<tokens::Chunk<Store>*>(dz + first) = {{c.x, c.y, c.z, c.w}};
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if (first + e < p.classes) dz[first + e] = T::rounded(d[e]);
            }
        });
        G::sync();  // the classes of the entries are written again below
        for (int k = t; k < p.entries; k += Group) {
            const int c = entry.cls[k];
            if (c >= 0) dz[c] = T::rounded(factor * (q(entry.logit[k]) - entry.share_of(c) / sums[0]));
        }
    }
    if constexpr (!Backward) {
        // last, under the gradient's stores
        const double log_mass = log(static_cast<double>(sums[0]));
        double terms = 0.0;
        for (int k = t; k < p.entries; k += Group) {
            const float e = entry.share[k];
            if (e == 0.0f) continue;
            const double log_p = (static_cast<double>(entry.teacher[k]) - top[0]) * p.per_t - log_mass;
            const double log_q = (static_cast<double>(entry.logit[k]) - m) * p.per_t - log_sum;
            terms += e * (log_p - log_q);
        }
        const float total = G::sum(static_cast<float>(terms), scratch);
        if (t == 0) p.loss[row] = static_cast<float>(weight * p.temperature * p.temperature * (total / sums[0]));
    }
}

template <typename T, int Group, int Held, bool Backward>
void launch_teams(const Params& p, hipStream_t stream) {
    constexpr int kTeams = Group < 256 ? 256 / Group : 1;
    const std::size_t lds = kTeams * 4 * sizeof(float) * static_cast<std::size_t>(Entries::round4(p.entries));
    constexpr int kThreads = Group < 256 ? 256 : Group;
    hipLaunchKernelGGL((distill_kernel<T, Group, Held, Backward>), tokens::grid_for(p.rows, kTeams, kThreads), dim3(kThreads),
                       lds, stream, p);
}

// The smallest team whose registers hold the row, 8 chunks a thread where that reaches: 4096 x 32768 bf16, loss and
// gradient, 121 us on 512 threads of 8 chunks, 131 on 256 of 16, 139 on 1024 of 4, 174 reading memory twice (a copy of the
// same bytes: 98 us).  Twice that: 2048 x 65536 131 us on 512 threads of 16 chunks, 169 on 1024 of 8, the gradient alone 130
// against 116.  Streaming such rows would be faster for the loss alone, which reads a row once either way (48 us against
// 62), but the loss would then differ in its last bits from the one that comes with the gradient.
template <typename T, bool Backward>
void launch(const Params& p, hipStream_t stream) {
    const int chunks = static_cast<int>(ceil_div(p.classes, T::kPerChunk));
    if (chunks <= 16 && p.entries <= 64) launch_teams<T, 16, 1, Backward>(p, stream);
    else if (chunks <= 32 && p.entries <= 64) launch_teams<T, 16, 2, Backward>(p, stream);
    else if (chunks <= 64 && p.entries <= 256) launch_teams<T, 64, 1, Backward>(p, stream);
    else if (chunks <= 128 && p.entries <= 256) launch_teams<T, 64, 2, Backward>(p, stream);
    else if (chunks <= 256 && p.entries <= 256) launch_teams<T, 64, 4, Backward>(p, stream);
    else if (chunks <= 512 && p.entries <= 256 && p.rows > 1024) launch_teams<T, 64, 8, Backward>(p, stream);
    else if (chunks <= 256 * 2) launch_teams<T, 256, 2, Backward>(p, stream);
    else if (chunks <= 256 * 4) launch_teams<T, 256, 4, Backward>(p, stream);
    else if (chunks <= 256 * 8) launch_teams<T, 256, 8, Backward>(p, stream);
    else if (chunks <= 512 * 8) launch_teams<T, 512, 8, Backward>(p, stream);
    else if (!Backward && chunks <= 512 * 16) launch_teams<T, 512, 16, false>(p, stream);
    else if (Backward && chunks <= 1024 * 8) launch_teams<T, 1024, 8, true>(p, stream);
    else if (chunks <= 1024 * 16) launch_teams<T, 1024, 16, Backward>(p, stream);
    else launch_teams<T, 1024, 0, Backward>(p, stream);
}

void run(Params& p, int type, bool backward, hipStream_t stream) {
    if (p.rows == 0) return;
    switch (type) {
        case tokens::kF32:
            backward ? launch<tokens::F32, true>(p, stream) : launch<tokens::F32, false>(p, stream);
            break;
        case tokens::kBf16:
            backward ? launch<tokens::Bf16, true>(p, stream) : launch<tokens::Bf16, false>(p, stream);
            break;
        default:
            backward ? launch<tokens::F16, true>(p, stream) : launch<tokens::F16, false>(p, stream);
    }
    check_launch("Launch distillation");
}

// The checks that both entry points share.
Params checked(const void* logits, int type, long long ld, const void* teacher, int teacher_type, const void* index,
               int index_bits, long long rows, int classes, int entries, double temperature, const void* dlogits,
               long long ldd) {
    require(tokens::known_type(type) && tokens::known_type(teacher_type),
            "Distillation takes logits of type 0 (fp32), 1 (bf16) or 3 (fp16).");
    require(index_bits == 32 || index_bits == 64, "Distillation takes indices of 32 or 64 bits.");
    require(rows >= 0 && classes > 0 && classes <= (1 << 24),
            "Distillation takes no negative number of rows and 1 to 2^24 classes.");
    require(entries > 0 && entries <= kMaxEntries, "Distillation takes 1 to 1024 teacher entries a row.");
    require(temperature > 0.0 && std::isfinite(temperature), "The distillation temperature must be positive and finite.");
    require(rows == 0 || (logits && teacher && index), "Distillation operands must be nonnull.");
    require(rows <= 1 || ld >= classes, "The rows of logits overlap.");
    require(!dlogits || rows <= 1 || ldd >= classes, "The rows of the gradient overlap.");
    const std::size_t size = tokens::type_size(type);
    require(aligned(logits, size) && aligned(dlogits, size) && aligned(teacher, tokens::type_size(teacher_type)) &&
                aligned(index, index_bits / 8),
            "Distillation operands must be aligned to their elements.");
    if (dlogits && rows > 0) {
        const char* a = static_cast<const char*>(logits);
        const char* b = static_cast<const char*>(dlogits);
        const bool apart = a + ((rows - 1) * ld + classes) * size <= b || b + ((rows - 1) * ldd + classes) * size <= a;
        require(apart || (a == b && (rows == 1 || ld == ldd)),
                "The gradient may take the place of the logits, or lie apart from them.");
    }
    Params p{};
    p.logits = logits;
    p.ld = ld;
    p.teacher = teacher;
    p.index = index;
    p.teacher_type = teacher_type;
    p.index_wide = index_bits == 64;
    p.rows = rows;
    p.classes = classes;
    p.entries = entries;
    p.temperature = temperature;
    p.per_t = 1.0 / temperature;
    p.rate = static_cast<float>(kLog2e / temperature);
    p.dlogits = const_cast<void*>(dlogits);
    p.ldd = ldd;
    return p;
}

}  // namespace distill
}  // namespace rl

RL_API int rl_distill_forward(const void* logits, int type, long long ld, const void* teacher_logits, int teacher_type,
                              const void* teacher_index, int index_bits, const float* weights, long long rows,
                              int classes, int entries, double temperature, float* loss_rows, float* lse,
                              void* dlogits, long long ld_dlogits, float grad_scale, void* stream) {
    return rl::guarded("rl_distill_forward", [&] {
        rl::distill::Params p = rl::distill::checked(logits, type, ld, teacher_logits, teacher_type, teacher_index,
                                                     index_bits, rows, classes, entries, temperature, dlogits, ld_dlogits);
        rl::require(rows == 0 || loss_rows, "Distillation writes the rows' losses: loss_rows is null.");
        rl::require(std::isfinite(grad_scale), "The gradient scale must be finite.");
        p.weights = weights;
        p.loss = loss_rows;
        p.lse_out = lse;
        p.grad_scale = grad_scale;
        rl::distill::run(p, type, false, rl::as_stream(stream));
    });
}

RL_API int rl_distill_backward(const void* logits, int type, long long ld, const void* teacher_logits, int teacher_type,
                               const void* teacher_index, int index_bits, const float* weights, const float* lse,
                               const float* dloss_rows, long long rows, int classes, int entries, double temperature,
                               void* dlogits, long long ld_dlogits, void* stream) {
    return rl::guarded("rl_distill_backward", [&] {
        rl::distill::Params p = rl::distill::checked(logits, type, ld, teacher_logits, teacher_type, teacher_index,
                                                     index_bits, rows, classes, entries, temperature, dlogits, ld_dlogits);
        rl::require(rows == 0 || (lse && dloss_rows && dlogits),
                    "The distillation gradient needs lse, the rows' loss gradients and an output.");
        p.weights = weights;
        p.lse_in = lse;
        p.dloss = dloss_rows;
        rl::distill::run(p, type, true, rl::as_stream(stream));
    });
}
