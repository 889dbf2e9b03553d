// Gated feed-forward products: h = act(x Wg^T) * (x Wu^T) and its backward pass.
//
// Forward, one kernel: the output tile's B operand is rows of both projections, so that a wave holds the gate and the
// up value of the same outputs in the same lane's accumulators; activation and product happen there and only h is
// written (4 R H I flops; x, both weights and h cross HBM once).
//
// Backward keeps nothing from the forward pass: the same kernel forms both projections again and its epilogue
// turns dh into dg = dh u act'(g), du = dh act(g) (4 R H I flops instead of writing and reading 8 R H bytes of fp32 gate
// and up values; 16-bit ones would be rounded twice).  Then dx = dg Wg + du Wu is one product over both halves of K and
// dW = [dg du]^T x one product of 2 H rows; dg and du are rounded to the operands' type once, as matrix operands have
// to be.
//
// fp32 operands take the three-piece bf16 products of gemm_split.hip and one pass for the gating.
#include "gemm.hpp"

#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

namespace rl {
namespace gated {

enum Activation : int { kSilu = 0, kGelu = 1, kRelu = 2 };

// act(g) and act'(g).
__device__ __forceinline__ void activate(float g, int kind, float& value, float& slope) {
    if (kind == kRelu) {
        value = g > 0.0f ? g : 0.0f;
        slope = g > 0.0f ? 1.0f : 0.0f;
    } else if (kind == kSilu) {
        const float s = 1.0f / (1.0f + __expf(-g));
        value = g * s;
        slope = s * (1.0f + g * (1.0f - s));
    } else {
        const float phi = 0.5f * erfcf(-0.70710678118654752440f * g);
        value = g * phi;
        slope = phi + g * (0.39894228040143267794f * __expf(-0.5f * g * g));
    }
}

// The 16-bit operand types.
struct Bf16 {
    typedef __bf16 Value;
    typedef __bf16 Fragment __attribute__((ext_vector_type(8)));
    __device__ __forceinline__ static gemm::f32x16_t mfma(Fragment a, Fragment b, gemm::f32x16_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
    __device__ __forceinline__ static unsigned short rounded(float v) { return f32_to_bf16_bits(v); }
    __device__ __forceinline__ static float value(unsigned short b) { return bf16_bits_to_f32(b); }
};
struct F16 {
    typedef _Float16 Value;
    typedef _Float16 Fragment __attribute__((ext_vector_type(8)));
    __device__ __forceinline__ static gemm::f32x16_t mfma(Fragment a, Fragment b, gemm::f32x16_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
    __device__ __forceinline__ static unsigned short rounded(float v) { return f32_to_f16_bits(v); }
    __device__ __forceinline__ static float value(unsigned short b) {
        return static_cast<float>(__builtin_bit_cast(_Float16, b));
    }
};

// ---------------------------------------------------------------------------
// The tile kernel: D[m, n] = sum_k A(m, k) B(n, k) on 16-bit operands
// ---------------------------------------------------------------------------
constexpr int kDepth = 64;  // K per LDS stage

// A product, its operands and what becomes of it.  K runs over `segments` pieces of k values each (dx: the gate and the
// up half), whose operands lie seg_a / seg_b elements apart.
struct Product {
    const unsigned short *a, *b;  // A(m, k): KC a[m lda + k], MN a[k lda + m]; B the same with n
    long long lda, ldb, seg_a, seg_b;
    int m, n, k, segments;
    int splits, tiles_per_split;  // K tiles of kDepth
    // plain output: d (operand type) or d32; split partials [splits][m][n] in d32
    unsigned short* d;
    float* d32;
    long long ldd;
    // gated: B's rows n < n are the gate's and those `up` elements further the up projection's
    long long up;
    const unsigned short* dh;
    long long ld_dh;
    unsigned short* h;           // forward
    long long ld_h;
    unsigned short* dpre;        // backward: [m][2 pitch], the gate's half first; columns n .. pitch are zeroed
    long long pitch;
    int activation;
};

enum Epilogue : int { kPlain = 0, kForward = 1, kBackward = 2 };

typedef unsigned int u32x4 __attribute__((ext_vector_type(4), may_alias));

constexpr int kBufferWord3 = 0x00020000;  // raw dword access (gfx9 buffer descriptor word 3)
constexpr unsigned kNowhere = 0x80000000u;  // past every window: reads as zero
// Windows and offsets inside them stay below 2^31 bytes.
constexpr long long kMaxPitch = 1LL << 21;

// LDS slot of 16-byte chunk c of row r (K-contiguous stage, 128-byte rows): the 16 rows of one ds_read_b128 phase
// lie in 16 distinct bank groups.
__device__ __forceinline__ int chunk_slot(int r, int c) { return c ^ ((r >> 1) & 7); }
// The same for granule c of K row k of an M/N-contiguous stage, read transposed.
__device__ __forceinline__ int granule_slot(int k, int c) { return c ^ (4 * (k & 3)); }

// Copies one K tile of an operand (Rows x kDepth) into LDS by DMA, 1 KiB an instruction.
template <bool MN, int Rows, int Waves>
struct Loader {
    static constexpr int kInstructions = Rows * kDepth * 2 / 1024;
    static_assert(kInstructions % Waves == 0, "whole instructions a wave");
    static constexpr int kPerWave = kInstructions / Waves;
    unsigned offset[kPerWave];
    int chunk[kPerWave];  // K-contiguous: first k of the lane's piece

    __device__ __forceinline__ void init(long long ld, int wave, int lane, bool halves) {
#pragma unroll
        for (int j = 0; j < kPerWave; ++j) {
            const int q = wave * kPerWave + j;
            if constexpr (MN) {
                constexpr int kGranules = Rows / 8;
                const int k = q * (64 / kGranules) + lane / kGranules;
                offset[j] = static_cast<unsigned>((k * ld + granule_slot(k, lane % kGranules) * 8) * 2);
                chunk[j] = 0;
            } else {
                const int row = q * 8 + lane / 8;
                chunk[j] = chunk_slot(row, lane % 8) * 8;
                // halves: 32 rows of the gate, then the same 32 of the up projection (whose window is another)
                const int source = halves ? (row / 64) * 32 + row % 32 : row;
                offset[j] = static_cast<unsigned>((source * ld + chunk[j]) * 2);
            }
        }
    }

    // base: the window's first element; rows, depth: what of the tile lies inside the operand
    __device__ __forceinline__ void fetch(const unsigned short* base, const unsigned short* other, long long ld, int rows,
                                          int depth, unsigned short* stage, int wave) const {
        // whole 16-byte pieces: what a K-contiguous row holds up to its next multiple of 8 is zero
        const long long bytes = MN ? ((depth - 1) * ld + rows) * 2 : ((rows - 1) * ld + (depth + 7) / 8 * 8) * 2;
        const int extent = rows > 0 && depth > 0 ? static_cast<int>(bytes) : 0;
#pragma unroll
        for (int j = 0; j < kPerWave; ++j) {
            const int q = wave * kPerWave + j;
            // the up projection's rows: every second 32 of the tile, 4 instructions
            const bool second = other && (q / 4) % 2;
            const __amdgpu_buffer_rsrc_t window = __builtin_amdgcn_make_buffer_rsrc(
                const_cast<unsigned short*>(second ? other : base), (short)0, extent, kBufferWord3);
            unsigned at = offset[j];
            if (!MN && depth < kDepth) at = chunk[j] < depth ? at : kNowhere;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                window, (__attribute__((address_space(3))) void*)(stage + q * 512), 16, at, 0, 0, 0);
        }
    }
};

// Waits for this wave's DMA, then for everyone's: the stage is complete, and the other one free.
__device__ __forceinline__ void stage_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <typename T, bool MN, int Rows, int N>
__device__ __forceinline__ void fragments(const unsigned short* stage, int first, int s, int lane,
                                          typename T::Fragment (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if constexpr (MN) {
            // the transposing read gives lane l of 16 the M offset l and four K rows: lane l addresses K row l / 4
            // of them, M offset 4 (l % 4)
            typedef short s16x4 __attribute__((ext_vector_type(4)));
            s16x4 part[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int k = 16 * s + 8 * (lane / 32) + 4 * r + (lane % 16) / 4;
                const int granule = (first + 32 * i) / 8 + 2 * ((lane / 16) % 2) + (lane % 4) / 2;
                const unsigned short* p = stage + k * Rows + granule_slot(k, granule) * 8 + 4 * (lane % 2);
                part[r] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
            }
            f[i] = __builtin_bit_cast(typename T::Fragment,
                                      __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            const int row = first + 32 * i + lane % 32;
            f[i] = *reinterpret_cast<const typename T::Fragment*>(stage + row * kDepth +
                                                                   chunk_slot(row, 2 * s + lane / 32) * 8);
        }
    }
}

// Workgroup b of the launch -> tile: consecutive tiles share operand panels, and each XCD (workgroups go to the 8 of
// them in turn) takes a contiguous run of tiles, walked in groups of 4 M tiles.
__device__ __forceinline__ void tile_of(int tiles_m, int tiles_n, int& tm, int& tn, int& split) {
    const int total = static_cast<int>(gridDim.x), b = static_cast<int>(blockIdx.x);
    const int whole = total / 8 * 8;
    const int id = b < whole ? (b % 8) * (total / 8) + b / 8 : b;
    constexpr int kGroup = 4;
    const int slice = tiles_m * tiles_n;
    split = id / slice;
    const int t = id % slice;
    const int first = t / (kGroup * tiles_n) * kGroup;
    const int group = min(tiles_m - first, kGroup);
    const int local = t % (kGroup * tiles_n);
    tm = first + local % group;
    tn = local / group;
}

template <typename T, bool AMN, bool BMN, int TM, int TN, int WavesM, int WavesN, int Out>
__global__ __launch_bounds__(WavesM * WavesN * kWave, 1) void product_kernel(Product p, int tiles_m, int tiles_n) {
    constexpr int kWaves = WavesM * WavesN;
    constexpr int kThreadCount = kWaves * kWave;
    constexpr int MI = TM / WavesM / 32, NJ = TN / WavesN / 32;
    constexpr bool kGated = Out != kPlain;
    static_assert(!kGated || (!AMN && !BMN && NJ == 2), "a wave's two column blocks are the gate's and the up's");
    constexpr int kOutN = kGated ? TN / 2 : TN;  // output columns of a tile
    constexpr int kStage = (TM + TN) * kDepth;
    // two objects: the compiler then tells reads of one stage from the DMA into the other
    __shared__ __attribute__((aligned(1024))) unsigned short stage0[kStage];
    __shared__ __attribute__((aligned(1024))) unsigned short stage1[kStage];

    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    const int lane = static_cast<int>(threadIdx.x) % kWave;
    const int wm = wave / WavesN, wn = wave % WavesN;
    int tm, tn, split;
    tile_of(tiles_m, tiles_n, tm, tn, split);
    const int m0 = tm * TM, n0 = tn * kOutN;
    const int rows_a = min(TM, p.m - m0), rows_b = min(kOutN, p.n - n0);

    Loader<AMN, TM, kWaves> la;
    Loader<BMN, TN, kWaves> lb;
    la.init(p.lda, wave, lane, false);
    lb.init(p.ldb, wave, lane, kGated);

    const int per_segment = (p.k + kDepth - 1) / kDepth;
    const int first_tile = split * p.tiles_per_split;
    const int last_tile = min(first_tile + p.tiles_per_split, per_segment * p.segments);
    int segment = first_tile / per_segment, k0 = (first_tile % per_segment) * kDepth;
    const auto fetch = [&](unsigned short* stage) {
        const int depth = min(kDepth, p.k - k0);
        const unsigned short* a = p.a + segment * p.seg_a + (AMN ? k0 * p.lda + m0 : m0 * p.lda + k0);
        const unsigned short* b = p.b + segment * p.seg_b + (BMN ? k0 * p.ldb + n0 : n0 * p.ldb + k0);
        // M/N-contiguous rows may be read up to their next multiple of 8, which the pitch covers
        la.fetch(a, nullptr, p.lda, AMN ? (rows_a + 7) / 8 * 8 : rows_a, depth, stage, wave);
        lb.fetch(b, kGated ? b + p.up : nullptr, p.ldb, BMN ? (rows_b + 7) / 8 * 8 : rows_b, depth,
                 stage + TM * kDepth, wave);
        k0 += kDepth;
        if (k0 >= p.k) k0 = 0, ++segment;
    };

    gemm::f32x16_t acc[MI][NJ];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.0f;

    const auto multiply = [&](const unsigned short* stage) {
#pragma unroll
        for (int s = 0; s < kDepth / 16; ++s) {
            typename T::Fragment a[MI], b[NJ];
            fragments<T, AMN, TM, MI>(stage, wm * (TM / WavesM), s, lane, a);
            fragments<T, BMN, TN, NJ>(stage + TM * kDepth, wn * (TN / WavesN), s, lane, b);
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NJ; ++j) acc[i][j] = T::mfma(a[i], b[j], acc[i][j]);
        }
    };

    if (first_tile < last_tile) fetch(stage0);
    for (int kt = first_tile; kt < last_tile; kt += 2) {
        stage_barrier();
        if (kt + 1 < last_tile) fetch(stage1);
        multiply(stage0);
        if (kt + 1 >= last_tile) break;
        stage_barrier();
        if (kt + 2 < last_tile) fetch(stage0);
        multiply(stage1);
    }

    // accumulator element v of lane l: column l % 32, row 8 (v / 4) + 4 (l / 32) + v % 4 of its 32 x 32 block
    const int col = lane % 32, row4 = 4 * (lane / 32);
    if constexpr (!kGated) {
        if (p.d32) {
            float* d = p.d32 + (p.splits > 1 ? static_cast<long long>(split) * p.m * p.n : 0);
            const long long ldd = p.splits > 1 ? p.n : p.ldd;
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    const int c = n0 + wn * (TN / WavesN) + 32 * j + col;
                    if (c >= p.n) continue;
#pragma unroll
                    for (int v = 0; v < 16; ++v) {
                        const int r = m0 + wm * (TM / WavesM) + 32 * i + 8 * (v / 4) + row4 + v % 4;
                        if (r < p.m) d[r * ldd + c] = acc[i][j][v];
                    }
                }
            return;
        }
    }

    // 16-bit outputs leave through LDS, whole tile rows at a time: in MI passes of 32 rows from each row of waves
    constexpr int kPitch = kOutN + 8;
    constexpr int kPassRows = 32 * WavesM;
    static_assert(kPassRows * kPitch <= kStage, "a pass fits a stage");
    constexpr int kChunks = kOutN / 8;  // 16-byte pieces of a tile row
    // between LDS and rows of `out` whose first `columns` values exist
    const auto move = [&](unsigned short* lds, unsigned short* out, long long ld, int columns, int pass, auto store) {
        const bool wide = reinterpret_cast<std::uintptr_t>(out) % 16 == 0 && ld % 8 == 0;
        for (int q = static_cast<int>(threadIdx.x); q < kPassRows * kChunks; q += kThreadCount) {
            const int local = q / kChunks, c = n0 + q % kChunks * 8;
            const int r = m0 + local / 32 * (TM / WavesM) + 32 * pass + local % 32;
            if (r >= p.m || c >= columns) continue;
            unsigned short* in = lds + local * kPitch + q % kChunks * 8;
            unsigned short* to = out + r * ld + c;
            if (wide && c + 8 <= columns) {
                u32x4& from = *reinterpret_cast<u32x4*>(in);
                u32x4& there = *reinterpret_cast<u32x4*>(to);
                if constexpr (decltype(store)::value) there = from;
                else from = there;
            } else {
                for (int e = 0; e < 8 && c + e < columns; ++e) {
                    if constexpr (decltype(store)::value) to[e] = in[e];
                    else in[e] = to[e];
                }
            }
        }
    };
    unsigned short *one = stage0, *two = stage1;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
        __syncthreads();  // the stages are free, and the pass before has left
        if constexpr (Out == kBackward) {
            move(one, const_cast<unsigned short*>(p.dh), p.ld_dh, p.n, i, std::false_type{});
            __syncthreads();
        }
#pragma unroll
        for (int v = 0; v < 16; ++v) {
            unsigned short* lds_one = one + (wm * 32 + 8 * (v / 4) + row4 + v % 4) * kPitch + col;
            if constexpr (!kGated) {
#pragma unroll
                for (int j = 0; j < NJ; ++j) lds_one[wn * (TN / WavesN) + 32 * j] = T::rounded(acc[i][j][v]);
            } else {
                lds_one += wn * 32;
                const float up = acc[i][1][v];
                float value, slope;
                activate(acc[i][0][v], p.activation, value, slope);
                if constexpr (Out == kForward) {
                    *lds_one = T::rounded(value * up);
                } else {
                    // columns past the last are zero, and so is what leaves for them
                    const float dh = n0 + wn * 32 + col < p.n ? T::value(*lds_one) : 0.0f;
                    *lds_one = T::rounded(dh * up * slope);
                    two[lds_one - one] = T::rounded(dh * value);
                }
            }
        }
        __syncthreads();
        if constexpr (Out == kPlain) {
            move(one, p.d, p.ldd, p.n, i, std::true_type{});
        } else if constexpr (Out == kForward) {
            move(one, p.h, p.ld_h, p.n, i, std::true_type{});
        } else {
            move(one, p.dpre, 2 * p.pitch, static_cast<int>(p.pitch), i, std::true_type{});
            move(two, p.dpre + p.pitch, 2 * p.pitch, static_cast<int>(p.pitch), i, std::true_type{});
        }
    }
}

template <typename T, bool AMN, bool BMN, int TM, int TN, int WavesM, int WavesN, int Out>
void launch_tiles(const Product& p, hipStream_t stream) {
    constexpr int kOutN = Out == kPlain ? TN : TN / 2;
    const long long tiles_m = ceil_div(p.m, TM), tiles_n = ceil_div(p.n, kOutN);
    require(tiles_m * tiles_n * p.splits <= INT_MAX, "The gated product has too many tiles.");
    hipLaunchKernelGGL((product_kernel<T, AMN, BMN, TM, TN, WavesM, WavesN, Out>),
                       dim3(static_cast<unsigned>(tiles_m * tiles_n * p.splits)), dim3(WavesM * WavesN * kWave), 0, stream,
                       p, static_cast<int>(tiles_m), static_cast<int>(tiles_n));
    check_launch("Launch gated product");
}

template <typename T, bool AMN, bool BMN, int Out>
void launch(const Product& p, hipStream_t stream) {
    launch_tiles<T, AMN, BMN, 128, 128, 2, 2, Out>(p, stream);
}

// dst[r, 0 .. pitch) = src[r, 0 .. columns), zeros after them: rows that the DMA can read in 16-byte pieces.
__global__ __launch_bounds__(256) void pack_kernel(const unsigned short* src, long long ld, long long rows, int columns,
                                                   unsigned short* dst, int pitch) {
    const long long pieces = rows * (pitch / 8);
    for (long long q = blockIdx.x * 256LL + threadIdx.x; q < pieces; q += gridDim.x * 256LL) {
        const long long r = q / (pitch / 8);
        const int c = static_cast<int>(q % (pitch / 8)) * 8;
        unsigned w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const unsigned short* s = src + r * ld + c + 2 * e;
            const unsigned lo = c + 2 * e < columns ? s[0] : 0u, hi = c + 2 * e + 1 < columns ? s[1] : 0u;
            w[e] = lo | (hi << 16);
        }
        *reinterpret_cast<u32x4*>(dst + r * pitch + c) = u32x4{w[0], w[1], w[2], w[3]};
    }
}

// fp32: gate and up [rows, hidden] of `pre` -> h
__global__ __launch_bounds__(256) void gate_forward(const float* pre, float* h, long long ld_h, long long rows, int hidden,
                                                    int activation) {
    const long long n = rows * hidden;
    for (long long q = blockIdx.x * 256LL + threadIdx.x; q < n; q += gridDim.x * 256LL) {
        float value, slope;
        activate(pre[q], activation, value, slope);
        h[q / hidden * ld_h + q % hidden] = value * pre[n + q];
    }
}

// fp32: gate and up of `pre` become their gradients.
__global__ __launch_bounds__(256) void gate_backward(float* pre, const float* dh, long long ld_dh, long long rows,
                                                     int hidden, int activation) {
    const long long n = rows * hidden;
    for (long long q = blockIdx.x * 256LL + threadIdx.x; q < n; q += gridDim.x * 256LL) {
        float value, slope;
        activate(pre[q], activation, value, slope);
        const float d = dh[q / hidden * ld_dh + q % hidden];
        const float up = pre[n + q];
        pre[q] = d * up * slope;
        pre[n + q] = d * value;
    }
}

// The splits' partial products in their order.
template <typename T>
__global__ __launch_bounds__(256) void reduce_kernel(const float* partial, int splits, long long m, int n,
                                                     unsigned short* d, float* d32, long long ldd) {
    const long long total = m * n;
    for (long long q = blockIdx.x * 256LL + threadIdx.x; q < total; q += gridDim.x * 256LL) {
        float sum = 0.0f;
        for (int s = 0; s < splits; ++s) sum += partial[s * total + q];
        const long long at = q / n * ldd + q % n;
        if (d32) d32[at] = sum;
        else d[at] = T::rounded(sum);
    }
}

__global__ __launch_bounds__(256) void clear_kernel(unsigned short* x, long long n) {
    for (long long q = blockIdx.x * 256LL + threadIdx.x; q < n; q += gridDim.x * 256LL) x[q] = 0;
}

unsigned blocks_for(long long items) { return static_cast<unsigned>(std::min<long long>((items + 255) / 256, 4096)); }

// ---------------------------------------------------------------------------
// Workspaces and calls
// ---------------------------------------------------------------------------
constexpr long long align8(long long v) { return (v + 7) / 8 * 8; }
constexpr std::size_t kAlign = 256;
constexpr std::size_t aligned_bytes(std::size_t b) { return (b + kAlign - 1) / kAlign * kAlign; }

struct Sizes {
    int type;
    long long rows;
    int inputs, hidden;
};

// K splits of a product with too few tiles: at least 256 workgroups, each with 8 K tiles of 64.
int split_tiles(long long m, long long n, long long k_tiles) {
    const long long tiles = static_cast<long long>(ceil_div(m, 128)) * ceil_div(n, 128);
    long long splits = 1;
    while (tiles * splits < 256 && k_tiles / (2 * splits) >= 8 && splits < 64) splits *= 2;
    return static_cast<int>(splits);
}

struct Layout {
    std::size_t x, w, dpre, partial, bytes;
};

// Where the parts of a 16-bit call's workspace lie.  Copies of x and w are counted always: whether they are needed goes
// by the addresses too.
Layout layout_of(const Sizes& s, bool backward) {
    Layout l{};
    std::size_t at = 0;
    const auto take = [&](long long elements, int size) {
        const std::size_t here = at;
        at += aligned_bytes(static_cast<std::size_t>(elements) * size);
        return here;
    };
    const long long pitch = align8(s.inputs), hidden_pitch = align8(s.hidden);
    l.x = take(s.rows * pitch, 2);
    l.w = take(2LL * s.hidden * pitch, 2);
    if (backward) {
        l.dpre = take(s.rows * 2 * hidden_pitch, 2);
        const int dx_splits = split_tiles(s.rows, s.inputs, 2 * ceil_div(s.hidden, kDepth));
        const int dw_splits = split_tiles(s.hidden, s.inputs, ceil_div(s.rows, kDepth));
        const long long dx = dx_splits > 1 ? dx_splits * s.rows * s.inputs : 0;
        const long long dw = dw_splits > 1 ? dw_splits * static_cast<long long>(s.hidden) * s.inputs : 0;
        l.partial = take(std::max(dx, dw), 4);
    }
    l.bytes = at;
    return l;
}

// K splits of the fp32 weight gradient: as the framework splits its own.
int fp32_splits(long long m, long long n, long long k) {
    const long long tiles = static_cast<long long>(ceil_div(m, 128)) * ceil_div(n, 128) * 2;
    int splits = 1;
    while (tiles * splits < 512 && splits * 2 <= k / 384 && splits < 64) splits *= 2;
    return splits;
}

std::size_t fp32_bytes(const Sizes& s, bool backward) {
    std::size_t bytes = aligned_bytes(static_cast<std::size_t>(2 * s.rows * s.hidden) * 4);
    if (backward) {
        const int splits = fp32_splits(s.hidden, s.inputs, s.rows);
        if (splits > 1) bytes += aligned_bytes(static_cast<std::size_t>(splits) * 2 * s.hidden * s.inputs * 4);
    }
    return bytes;
}

std::size_t workspace_bytes(const Sizes& s, bool backward) {
    return s.type == 0 ? fp32_bytes(s, backward) : layout_of(s, backward).bytes;
}

struct Operands {
    const void *x, *w, *dh;
    void *h, *dx, *dw;
    long long ldx, ld_h, ld_dh, ld_dx;
    int activation, dw_fp32;
    char* workspace;
};

void run_fp32(const Sizes& s, const Operands& o, bool backward, hipStream_t stream) {
    const int rows = static_cast<int>(s.rows), in = s.inputs, hidden = s.hidden;
    const float *x = static_cast<const float*>(o.x), *w = static_cast<const float*>(o.w);
    float* pre = reinterpret_cast<float*>(o.workspace);
    const long long each = s.rows * hidden, weights = static_cast<long long>(hidden) * in;
    run_gemm(2, 0, 0, 1, 1, rows, hidden, in, 2, x, o.ldx, 0, w, in, weights, nullptr, pre, hidden, each, nullptr, 0, 0.0f,
             0, 1, nullptr, 0, stream, nullptr, nullptr, nullptr);
    if (!backward) {
        hipLaunchKernelGGL(gate_forward, dim3(blocks_for(each)), dim3(256), 0, stream, pre, static_cast<float*>(o.h), o.ld_h,
                           s.rows, hidden, o.activation);
        check_launch("Launch gating");
        return;
    }
    hipLaunchKernelGGL(gate_backward, dim3(blocks_for(each)), dim3(256), 0, stream, pre, static_cast<const float*>(o.dh),
                       o.ld_dh, s.rows, hidden, o.activation);
    check_launch("Launch gating gradient");
    if (o.dx) {
        float* dx = static_cast<float*>(o.dx);
        for (int half = 0; half < 2; ++half)
            run_gemm(2, 0, 0, 1, 0, rows, in, hidden, 1, pre + half * each, hidden, 0, w + half * weights, in, 0,
                     half ? dx : nullptr, dx, o.ld_dx, 0, nullptr, 0, half ? 1.0f : 0.0f, 0, 1, nullptr, 0, stream, nullptr,
                     nullptr, nullptr);
    }
    if (o.dw) {
        const int splits = fp32_splits(hidden, in, s.rows);
        char* partial = o.workspace + aligned_bytes(static_cast<std::size_t>(2 * each) * 4);
        run_gemm(2, 0, 0, 0, 0, hidden, in, rows, 2, pre, hidden, each, x, o.ldx, 0, nullptr, static_cast<float*>(o.dw), in,
                 weights, nullptr, 0, 0.0f, 0, splits, splits > 1 ? reinterpret_cast<float*>(partial) : nullptr,
                 splits > 1 ? static_cast<std::size_t>(splits) * 2 * weights * 4 : 0, stream, nullptr, nullptr, nullptr);
    }
}

template <typename T, bool AMN, bool BMN>
void run_plain(Product p, int splits, float* partial, hipStream_t stream) {
    const int tiles = static_cast<int>(ceil_div(p.k, kDepth)) * p.segments;
    p.tiles_per_split = static_cast<int>(ceil_div(tiles, splits));
    p.splits = static_cast<int>(ceil_div(tiles, p.tiles_per_split));
    if (p.splits <= 1) {
        launch<T, AMN, BMN, kPlain>(p, stream);
        return;
    }
    Product parts = p;
    parts.d = nullptr;
    parts.d32 = partial;
    launch<T, AMN, BMN, kPlain>(parts, stream);
    hipLaunchKernelGGL((reduce_kernel<T>), dim3(blocks_for(static_cast<long long>(p.m) * p.n)), dim3(256), 0, stream, partial,
                       p.splits, static_cast<long long>(p.m), p.n, p.d, p.d32, p.ldd);
    check_launch("Launch gated product reduction");
}

// The operand as the DMA reads it: in place, or copied to rows of 16-byte pieces.
const unsigned short* readable(const void* data, long long rows, int columns, long long& ld, char* space,
                               hipStream_t stream) {
    const unsigned short* p = static_cast<const unsigned short*>(data);
    if (aligned(p, 16) && columns % 8 == 0 && (ld % 8 == 0 || rows == 1) && ld <= kMaxPitch) {
        if (rows == 1) ld = align8(columns);
        return p;
    }
    unsigned short* copy = reinterpret_cast<unsigned short*>(space);
    const int pitch = static_cast<int>(align8(columns));
    hipLaunchKernelGGL(pack_kernel, dim3(blocks_for(rows * (pitch / 8))), dim3(256), 0, stream, p, ld, rows, columns, copy,
                       pitch);
    check_launch("Launch operand copy");
    ld = pitch;
    return copy;
}

template <typename T>
void run_16bit(const Sizes& s, const Operands& o, bool backward, hipStream_t stream) {
    const Layout l = layout_of(s, backward);
    long long ldx = o.ldx, ldw = s.inputs;
    const unsigned short* x = readable(o.x, s.rows, s.inputs, ldx, o.workspace + l.x, stream);
    const unsigned short* w = readable(o.w, 2LL * s.hidden, s.inputs, ldw, o.workspace + l.w, stream);
    Product p{};
    p.a = x;
    p.lda = ldx;
    p.b = w;
    p.ldb = ldw;
    p.up = s.hidden * ldw;
    p.m = static_cast<int>(s.rows);
    p.n = s.hidden;
    p.k = static_cast<int>(align8(s.inputs));
    p.segments = 1;
    p.splits = 1;
    p.tiles_per_split = static_cast<int>(ceil_div(p.k, kDepth));
    p.activation = o.activation;
    p.h = static_cast<unsigned short*>(o.h);
    p.ld_h = o.ld_h;
    if (!backward) {
        launch<T, false, false, kForward>(p, stream);
        return;
    }
    const long long pitch = align8(s.hidden);
    unsigned short* dpre = reinterpret_cast<unsigned short*>(o.workspace + l.dpre);
    float* partial = reinterpret_cast<float*>(o.workspace + l.partial);
    p.dh = static_cast<const unsigned short*>(o.dh);
    p.ld_dh = o.ld_dh;
    p.dpre = dpre;
    p.pitch = pitch;
    launch<T, false, false, kBackward>(p, stream);
    if (o.dx) {
        Product q{};
        q.a = dpre;
        q.lda = 2 * pitch;
        q.seg_a = pitch;
        q.b = w;
        q.ldb = ldw;
        q.seg_b = s.hidden * ldw;
        q.m = static_cast<int>(s.rows);
        q.n = s.inputs;
        q.k = s.hidden;
        q.segments = 2;
        q.d = static_cast<unsigned short*>(o.dx);
        q.ldd = o.ld_dx;
        run_plain<T, false, true>(q, split_tiles(s.rows, s.inputs, 2 * ceil_div(s.hidden, kDepth)), partial, stream);
    }
    if (o.dw) {
        for (int half = 0; half < 2; ++half) {
            Product q{};
            q.a = dpre + half * pitch;
            q.lda = 2 * pitch;
            q.b = x;
            q.ldb = ldx;
            q.m = s.hidden;
            q.n = s.inputs;
            q.k = static_cast<int>(s.rows);
            q.segments = 1;
            q.ldd = s.inputs;
            const long long to = half * static_cast<long long>(s.hidden) * s.inputs;
            if (o.dw_fp32) q.d32 = static_cast<float*>(o.dw) + to;
            else q.d = static_cast<unsigned short*>(o.dw) + to;
            run_plain<T, true, true>(q, split_tiles(s.hidden, s.inputs, ceil_div(s.rows, kDepth)), partial, stream);
        }
    }
}

void check_sizes(const Sizes& s) {
    require(s.type == 0 || s.type == 1 || s.type == 3, "Gated products take operands of type 0 (fp32), 1 (bf16) or 3 (fp16).");
    require(s.rows >= 0 && s.rows <= (1 << 24) && s.inputs > 0 && s.hidden > 0 && s.inputs <= (1 << 20) &&
                s.hidden <= (1 << 20),
            "Gated products take 0 to 2^24 rows and 1 to 2^20 inputs and hidden values.");
    require(static_cast<long long>(s.inputs) * s.hidden <= INT_MAX && s.rows * s.hidden <= INT_MAX &&
                s.rows * s.inputs <= INT_MAX,
            "A gated product's matrices hold at most 2^31 - 1 values each.");
}

void run(const Sizes& s, const Operands& o, std::size_t bytes, bool backward, hipStream_t stream) {
    check_sizes(s);
    require(o.activation >= kSilu && o.activation <= kRelu, "Unknown activation: 0 silu, 1 gelu, 2 relu.");
    const std::size_t need = workspace_bytes(s, backward);
    require(s.rows == 0 || need == 0 || (o.workspace && bytes >= need && aligned(o.workspace, 16)),
            "The gated workspace is null, misaligned or too small (rl_gated_workspace).");
    const int size = s.type == 0 ? 4 : 2;
    for (const void* q : {o.x, o.w, o.dh, static_cast<const void*>(o.h), static_cast<const void*>(o.dx)})
        require(aligned(q, size), "Gated operands must be aligned to their elements.");
    require(aligned(o.dw, o.dw_fp32 ? 4 : size), "Gated operands must be aligned to their elements.");
    require(s.rows <= 1 || (o.ldx >= s.inputs && (!o.h || o.ld_h >= s.hidden) && (!o.dh || o.ld_dh >= s.hidden) &&
                            (!o.dx || o.ld_dx >= s.inputs)),
            "The rows of a gated operand overlap.");
    if (s.rows == 0) {
        if (backward && o.dw) {  // a sum of nothing
            const long long halves = 2LL * s.hidden * s.inputs * (s.type == 0 || o.dw_fp32 ? 2 : 1);
            hipLaunchKernelGGL(clear_kernel, dim3(blocks_for(halves)), dim3(256), 0, stream,
                               static_cast<unsigned short*>(o.dw), halves);
            check_launch("Launch gradient clearing");
        }
        return;
    }
    if (s.type == 0) run_fp32(s, o, backward, stream);
    else if (s.type == 1) run_16bit<Bf16>(s, o, backward, stream);
    else run_16bit<F16>(s, o, backward, stream);
}

}  // namespace gated
}  // namespace rl

RL_API size_t rl_gated_workspace(int type, long long rows, int inputs, int hidden, int backward) {
    std::size_t bytes = 0;
    rl::guarded("rl_gated_workspace", [&] {
        const rl::gated::Sizes s{type, rows, inputs, hidden};
        rl::gated::check_sizes(s);
        bytes = rows ? rl::gated::workspace_bytes(s, backward != 0) : 0;
    });
    return bytes;
}

RL_API int rl_gated_forward(int type, long long rows, int inputs, int hidden, int activation, const void* x, long long ldx,
                            const void* w, void* h, long long ld_h, void* workspace, size_t workspace_bytes, void* stream) {
    return rl::guarded("rl_gated_forward", [&] {
        rl::require(rows == 0 || (x && w && h), "Gated operands must be nonnull.");
        rl::gated::Operands o{};
        o.x = x, o.w = w, o.h = h, o.ldx = ldx, o.ld_h = ld_h, o.activation = activation;
        o.workspace = static_cast<char*>(workspace);
        rl::gated::run({type, rows, inputs, hidden}, o, workspace_bytes, false, rl::as_stream(stream));
    });
}

RL_API int rl_gated_backward(int type, long long rows, int inputs, int hidden, int activation, const void* x, long long ldx,
                             const void* w, const void* dh, long long ld_dh, void* dx, long long ld_dx, void* dw, int dw_fp32,
                             void* workspace, size_t workspace_bytes, void* stream) {
    return rl::guarded("rl_gated_backward", [&] {
        rl::require(dx || dw, "The gated backward pass has no output.");
        rl::require(rows == 0 || (x && w && dh), "Gated operands must be nonnull.");
        rl::gated::Operands o{};
        o.x = x, o.w = w, o.dh = dh, o.dx = dx, o.dw = dw, o.ldx = ldx, o.ld_dh = ld_dh, o.ld_dx = ld_dx;
        o.activation = activation, o.dw_fp32 = dw_fp32;
        o.workspace = static_cast<char*>(workspace);
        rl::gated::run({type, rows, inputs, hidden}, o, workspace_bytes, true, rl::as_stream(stream));
    });
}
