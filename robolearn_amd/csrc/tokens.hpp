// Rows of logits over discrete tokens: element types, and one row held by a group of threads.
#pragma once

#include "common.hpp"

namespace rl {
namespace tokens {

// Element types of logits, as the product modes number them.
enum Type : int { kF32 = 0, kBf16 = 1, kF16 = 3 };

inline bool known_type(int type) { return type == kF32 || type == kBf16 || type == kF16; }
inline int type_size(int type) { return type == kF32 ? 4 : 2; }

// Workgroups of `threads` for so many rows: a launch holds fewer than 2^32 threads.
inline dim3 grid_for(long long rows, int rows_a_group, int threads) {
    const long long groups = (rows - 1) / rows_a_group + 1;
    require(groups <= 0xffffffffLL / threads, "Too many rows for one launch.");
    return dim3(static_cast<unsigned>(groups));
}

struct F32 {
    typedef float Store;
    static constexpr int kPerChunk = 4;
    static constexpr unsigned kNegInf = 0xff800000u;  // -infinity in every element of a 32-bit word
    static constexpr int kKeyShift = 0;  // last bits in which the values, as fp32, cannot differ
    __device__ __forceinline__ static void unpack(const uint4& c, float (&v)[4]) {
        v[0] = __uint_as_float(c.x), v[1] = __uint_as_float(c.y);
        v[2] = __uint_as_float(c.z), v[3] = __uint_as_float(c.w);
    }
    __device__ __forceinline__ static uint4 pack(const float (&v)[4]) {
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
    __device__ __forceinline__ static float value(Store s) { return s; }
    __device__ __forceinline__ static Store rounded(float v) { return v; }
};

struct Bf16 {
    typedef unsigned short Store;
    static constexpr int kPerChunk = 8;
    static constexpr unsigned kNegInf = 0xff80ff80u;
    static constexpr int kKeyShift = 16;
    __device__ __forceinline__ static void unpack(const uint4& c, float (&v)[8]) {
        const unsigned w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    __device__ __forceinline__ static uint4 pack(const float (&v)[8]) {
        return make_uint4(f32x2_to_bf16x2(v[0], v[1]), f32x2_to_bf16x2(v[2], v[3]), f32x2_to_bf16x2(v[4], v[5]),
                          f32x2_to_bf16x2(v[6], v[7]));
    }
    __device__ __forceinline__ static float value(Store s) { return bf16_bits_to_f32(s); }
    __device__ __forceinline__ static Store rounded(float v) { return f32_to_bf16_bits(v); }
};

struct F16 {
    typedef unsigned short Store;
    static constexpr int kPerChunk = 8;
    static constexpr unsigned kNegInf = 0xfc00fc00u;
    static constexpr int kKeyShift = 13;
    __device__ __forceinline__ static void unpack(const uint4& c, float (&v)[8]) {
        const unsigned w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f16x2_t h = __builtin_bit_cast(f16x2_t, w[i]);
            v[2 * i] = static_cast<float>(h[0]);
            v[2 * i + 1] = static_cast<float>(h[1]);
        }
    }
    __device__ __forceinline__ static uint4 pack(const float (&v)[8]) {
        return make_uint4(f32x2_to_f16x2(v[0], v[1]), f32x2_to_f16x2(v[2], v[3]), f32x2_to_f16x2(v[4], v[5]),
                          f32x2_to_f16x2(v[6], v[7]));
    }
    __device__ __forceinline__ static float value(Store s) {
        return static_cast<float>(__builtin_bit_cast(_Float16, s));
    }
    __device__ __forceinline__ static Store rounded(float v) { return f32_to_f16_bits(v); }
};

// 16 bytes at any address that suits one element: rows of odd length start anywhere.
template <typename Store>
struct __attribute__((packed, aligned(sizeof(Store)))) Chunk {
    unsigned w[4];
};

// A group of Group threads that works on one row: 16 lanes of a wave, a wave, or a whole workgroup.
template <int Group>
struct Team {
    static constexpr bool kInWave = Group <= kWave;
    static constexpr int kWaves = kInWave ? 1 : Group / kWave;
    static_assert(Group == 16 || Group % kWave == 0, "a row of lanes or whole waves");

    __device__ __forceinline__ static int thread() { return static_cast<int>(threadIdx.x) % Group; }
    __device__ __forceinline__ static int wave() {
        return kInWave ? 0 : __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    }
    // Orders the group's memory accesses (a wave's own LDS operations execute in order).
    __device__ __forceinline__ static void sync() {
        if constexpr (kInWave) {
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
        } else {
            __syncthreads();
        }
    }
    // The group's sum, or maximum, of every value; every thread receives it.  scratch: N kWaves floats of LDS.
    template <int N>
    __device__ __forceinline__ static void sum(float (&v)[N], float* scratch) {
        reduce(v, scratch, [](float a, float b) { return a + b; }, [](float a) { return wave_sum(a); });
    }
    template <int N>
    __device__ __forceinline__ static void max(float (&v)[N], float* scratch) {
        reduce(v, scratch, [](float a, float b) { return fmaxf(a, b); }, [](float a) { return wave_max(a); });
    }
    __device__ __forceinline__ static float sum(float v, float* scratch) {
        float one[1] = {v};
        sum(one, scratch);
        return one[0];
    }
    __device__ __forceinline__ static float max(float v, float* scratch) {
        float one[1] = {v};
        max(one, scratch);
        return one[0];
    }

private:
    template <int N, typename Two, typename Wave>
    __device__ __forceinline__ static void reduce(float (&v)[N], float* scratch, Two two, Wave over_wave) {
        if constexpr (Group == 16) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                v[i] = two(v[i], dpp<kDppXor1>(v[i]));
                v[i] = two(v[i], dpp<kDppXor2>(v[i]));
                v[i] = two(v[i], dpp<kDppHalfMirror>(v[i]));
                v[i] = two(v[i], dpp<kDppMirror>(v[i]));
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = over_wave(v[i]);
            if constexpr (!kInWave) {
                __syncthreads();
                if (threadIdx.x % kWave == 0) {
#pragma unroll
                    for (int i = 0; i < N; ++i) scratch[i * kWaves + wave()] = v[i];
                }
                __syncthreads();
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    v[i] = scratch[i * kWaves];
#pragma unroll
                    for (int w = 1; w < kWaves; ++w) v[i] = two(v[i], scratch[i * kWaves + w]);
                }
            }
        }
    }
};

// A row of `classes` elements as 16-byte chunks: chunk t + i * Group belongs to thread t.  The last chunk may be
// partial; chunks and elements past the row read as -infinity.  Held > 0: the row stays in the registers of the
// group (Held chunks a thread); 0: every chunk() reads memory again.
template <typename T, int Group, int Held>
struct Row {
    typedef typename T::Store Store;
    static constexpr int V = T::kPerChunk;
    const Store* data;
    int full, rest;  // whole chunks, elements of the partial one
    uint4 held[Held > 0 ? Held : 1];

    __device__ __forceinline__ static uint4 nothing() {
        return make_uint4(T::kNegInf, T::kNegInf, T::kNegInf, T::kNegInf);
    }
    __device__ __forceinline__ uint4 load(int c) const {
        const Chunk<Store> x = *reinterpret_cast<const Chunk<Store>*>(data + static_cast<long long>(c) * V);
        return make_uint4(x.w[0], x.w[1], x.w[2], x.w[3]);
    }
    __device__ __forceinline__ uint4 load_rest() const {
        unsigned w[4] = {T::kNegInf, T::kNegInf, T::kNegInf, T::kNegInf};
        const Store* p = data + static_cast<long long>(full) * V;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            if (e >= rest) continue;
            if constexpr (V == 4) {
                w[e] = __builtin_bit_cast(unsigned, p[e]);
            } else {
                const unsigned bits = p[e];
                w[e / 2] = e % 2 ? (w[e / 2] & 0xffffu) | (bits << 16) : (w[e / 2] & 0xffff0000u) | bits;
            }
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }

    // chunk c of the row, from memory
    __device__ __forceinline__ uint4 read(int c) const {
        return c < full ? load(c) : c == full && rest ? load_rest() : nothing();
    }

    // passes over the row: chunk(i) for i < passes()
    __device__ __forceinline__ int passes() const { return (full + (rest ? 1 : 0) + Group - 1) / Group; }

    __device__ __forceinline__ void open(const Store* row, int classes) {
        data = row;
        full = classes / V;
        rest = classes % V;
        if constexpr (Held > 0) {
            const int t = Team<Group>::thread();
#pragma unroll
            for (int i = 0; i < Held; ++i) held[i] = t + i * Group < full ? load(t + i * Group) : nothing();
            if (rest && t == full % Group) {
                const uint4 last = load_rest();
#pragma unroll
                for (int i = 0; i < Held; ++i)
                    if (i == full / Group) held[i] = last;
            }
        }
    }

    __device__ __forceinline__ uint4 chunk(int i) const {
        if constexpr (Held > 0) return held[i];
        else return read(Team<Group>::thread() + i * Group);
    }

    // Makes the compiler unpack the held row again after this point, instead of holding its values in two or four times as
    // many registers.
    __device__ __forceinline__ void packed() {
        if constexpr (Held > 0) {
#pragma unroll
            for (int i = 0; i < Held; ++i)
                asm volatile("" : "+v"(held[i].x), "+v"(held[i].y), "+v"(held[i].z), "+v"(held[i].w));
        }
    }

    // f(i, values, index of the first value) for every pass
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        const int t = Team<Group>::thread();
        if constexpr (Held > 0) {
#pragma unroll
            for (int i = 0; i < Held; ++i) {
                float v[V];
                T::unpack(held[i], v);
                f(i, v, (t + i * Group) * V);
            }
        } else {
            const int n = passes();
#pragma unroll 4
            for (int i = 0; i < n; ++i) {
                float v[V];
                T::unpack(chunk(i), v);
                f(i, v, (t + i * Group) * V);
            }
        }
    }
};

// A long row over a whole workgroup: as Row, but the passes run in loops.  Held: the row lives in the registers of the
// group (up to kHeldChunks chunks a thread, four vectors that a loop indexes by one scalar); unrolled over 16 chunks the
// passes over it would not fit the instruction cache.  Else every pass reads memory again.
constexpr int kHeldChunks = 16;

template <typename T, int Group, bool Held>
struct LongRow {
    typedef typename T::Store Store;
    typedef unsigned Words __attribute__((ext_vector_type(kHeldChunks)));
    static constexpr int V = T::kPerChunk;
    Row<T, Group, 0> memory;
    Words x, y, z, w;

    __device__ __forceinline__ void open(const Store* row, int classes) {
        memory.open(row, classes);
        if constexpr (Held) {
            const int t = static_cast<int>(threadIdx.x);
#pragma unroll
            for (int i = 0; i < kHeldChunks; ++i) {
                const int c = t + i * Group;
                const uint4 q = c < memory.full ? memory.load(c) : memory.nothing();
                x[i] = q.x, y[i] = q.y, z[i] = q.z, w[i] = q.w;
            }
            if (memory.rest && t == memory.full % Group) {
                const uint4 q = memory.load_rest();
                const int last = memory.full / Group;
#pragma unroll
                for (int i = 0; i < kHeldChunks; ++i)
                    if (i == last) x[i] = q.x, y[i] = q.y, z[i] = q.z, w[i] = q.w;
            }
        }
    }
    __device__ __forceinline__ int passes() const { return memory.passes(); }
    __device__ __forceinline__ uint4 read(int c) const { return memory.read(c); }
    __device__ __forceinline__ uint4 chunk(int i) const {
        if constexpr (Held) return make_uint4(x[i], y[i], z[i], w[i]);
        else return memory.chunk(i);
    }
    __device__ __forceinline__ static float top_of(const float (&v)[V]) {
        float top = v[0];
#pragma unroll
        for (int e = 1; e < V; ++e) top = fmaxf(top, v[e]);
        return top;
    }
    // f(i, values, their maximum) for every pass
    template <typename F>
    __device__ __forceinline__ void each_pass(F f) const {
        const int n = passes();
#pragma unroll 1
        for (int i = 0; i < n; ++i) {
            float v[V];
            T::unpack(chunk(i), v);
            f(i, v, top_of(v));
        }
    }
    // f(values, index of the first)
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        const int n = passes();
#pragma unroll 1
        for (int i = 0; i < n; ++i) {
            float v[V];
            T::unpack(chunk(i), v);
            f(v, (static_cast<int>(threadIdx.x) + i * Group) * V);
        }
    }
    // the same where wanted(maximum) holds
    template <typename W, typename F>
    __device__ __forceinline__ void each_with(W wanted, F f) const {
        const int n = passes();
#pragma unroll 1
        for (int i = 0; i < n; ++i) {
            float v[V];
            T::unpack(chunk(i), v);
            if (wanted(top_of(v))) f(v, (static_cast<int>(threadIdx.x) + i * Group) * V);
        }
    }
    // f(maximum of the chunk)
    template <typename F>
    __device__ __forceinline__ void each_max(F f) const {
        const int n = passes();
        if constexpr (Held) {
#pragma unroll
            for (int i = 0; i < kHeldChunks; ++i) {
                float v[V];
                T::unpack(chunk(i), v);
                f(top_of(v));
            }
        } else {
#pragma unroll 4
            for (int i = 0; i < n; ++i) {
                float v[V];
                T::unpack(chunk(i), v);
                f(top_of(v));
            }
        }
    }
};

}  // namespace tokens
}  // namespace rl
