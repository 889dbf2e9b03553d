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
// What bounds the large sizes is the K loop: 8192 rows, 1024 inputs, 4096 hidden in bf16 take 127 us forward (1.08 PFLOP/s;
// a library product of the same sizes alone 116 us) and 385 us backward (1.07 PFLOP/s with the recomputation), the matrix
// cores busy 51 % of the cycles in the forward projection and 59 % in the gradients (the epilogues' VALU work, about a
// fifth of the cycles, overlaps only loads on tiles of 256: one workgroup a CU).  Small sizes are one chain of loads, products and
// stores behind the launch: see stream_kernel and the plans.
//
// fp32 operands take the three-piece bf16 products of gemm_split.hip and one pass for the gating (2048 x 256 x 1024
// backward 76 us: products of 19, 19 and 24 us, the pass 8 us at 5 TB/s, two sums of 5 us).
#include "gemm.hpp"

#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

RL_API std::size_t rl_gemm_workspace(int mode, int m, int n, int k, int batch, int splits) noexcept;

namespace rl {
namespace gated {

enum Activation : int { kSilu = 0, kGelu = 1, kRelu = 2 };

// act(g) and act'(g).  The reciprocals and powers of two are the hardware's (1 ulp).  gelu: with E = exp(-g^2 / 2), which
// the slope needs anyway, Phi(-|g|) = E P(1 / (1 + 0.4 |g| / sqrt 2)), P a polynomial of degree 8 fitted to
// erfcx(x) / 2 over 0 <= x <= 10 by iteratively weighted least squares: 4.3e-7 relative in fp32, tails included.
template <int Kind>
__device__ __forceinline__ void activate(float g, float& value, float& slope) {
    constexpr float kLog2e = 1.44269504088896340736f;
    if constexpr (Kind == kRelu) {
        value = g > 0.0f ? g : 0.0f;
        slope = g > 0.0f ? 1.0f : 0.0f;
    } else if constexpr (Kind == kSilu) {
        const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * g));
        value = g * s;
        slope = s * (1.0f + g * (1.0f - s));
    } else {
        const float e = __builtin_amdgcn_exp2f((-0.5f * kLog2e) * (g * g));
        const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.28284271247461900976f, fabsf(g), 1.0f));
        float q = 0.03533526510000229f;
        q = __builtin_fmaf(q, t, -0.1904902458190918f);
        q = __builtin_fmaf(q, t, 0.3330724537372589f);
        q = __builtin_fmaf(q, t, -0.18317051231861115f);
        q = __builtin_fmaf(q, t, 0.2072092741727829f);
        q = __builtin_fmaf(q, t, 0.06584122031927109f);
        q = __builtin_fmaf(q, t, 0.12010600417852402f);
        q = __builtin_fmaf(q, t, 0.1120610386133194f);
        q = __builtin_fmaf(q, t, 3.543297134456225e-05f) * e;
        const float phi = g >= 0.0f ? 1.0f - q : q;
        value = g * phi;
        slope = __builtin_fmaf(g, 0.39894228040143267794f * e, phi);
    }
}

// f(std::integral_constant<int, kind>) for the activation that runs.
template <typename F>
void with_activation(int kind, F f) {
    if (kind == kSilu) f(std::integral_constant<int, kSilu>{});
    else if (kind == kGelu) f(std::integral_constant<int, kGelu>{});
    else f(std::integral_constant<int, kRelu>{});
}

typedef float f32x4 __attribute__((ext_vector_type(4)));

// The 16-bit operand types.
struct Bf16 {
    typedef __bf16 Value;
    typedef __bf16 Fragment __attribute__((ext_vector_type(8)));
    __device__ __forceinline__ static gemm::f32x16_t mfma(Fragment a, Fragment b, gemm::f32x16_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
    __device__ __forceinline__ static f32x4 mfma16(Fragment a, Fragment b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
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
    __device__ __forceinline__ static f32x4 mfma16(Fragment a, Fragment b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
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
    // plain: rows 0 .. fold_to and fold .. fold + fold_to are the output's, one after the other, and the rest none (dW: the
    // gate's rows up to a multiple of 8, then the up projection's up to one)
    int fold, fold_to;
};

enum Epilogue : int { kPlain = 0, kForward = 1, kBackward = 2 };

// The output row of row r, -1 for none.
__device__ __forceinline__ long long folded(int r, int fold, int fold_to) {
    const int of_half = r >= fold ? r - fold : r;
    return of_half < fold_to ? (r >= fold ? of_half + fold_to : of_half) : -1;
}

typedef unsigned int u32x4 __attribute__((ext_vector_type(4), may_alias));

constexpr int kBufferWord3 = 0x00020000;  // raw dword access (gfx9 buffer descriptor word 3)
constexpr unsigned kNowhere = 0x80000000u;  // past every window: reads as zero
// Windows and offsets inside them stay below 2^31 bytes.
constexpr long long kMaxPitch = 1LL << 21;

// LDS slot of 16-byte chunk c of row r (K-contiguous stage, 128-byte rows): the 16 rows of one ds_read_b128 phase
// lie in 16 distinct bank groups.
__device__ __forceinline__ int chunk_slot(int r, int c) { return c ^ ((r >> 1) & 7); }
// The same for granule c of K row k of an M/N-contiguous stage of `Rows` values a K row, read transposed.
template <int Rows>
__device__ __forceinline__ int granule_slot(int k, int c) {
    return c ^ (4 * (k & 3) & (Rows / 8 - 1));
}

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
                offset[j] = static_cast<unsigned>((k * ld + granule_slot<Rows>(k, lane % kGranules) * 8) * 2);
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

// A barrier for what goes through LDS: this wave's LDS operations are done, its global stores (which __syncthreads would
// wait for) need not be.
__device__ __forceinline__ void lds_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// A wave's fragments of one operand: N blocks of 32 rows from row `first` of a stage (a multiple of 32), 16 K values a step.
template <typename T, bool MN, int Rows, int N>
struct Reader {
    int at[MN ? N : kDepth / 16];  // element offsets: the lane's of each block (MN), or of each step

    __device__ __forceinline__ void init(int first, int lane) {
        if constexpr (MN) {
            // the transposing read gives lane l of 16 the M offset l and four K rows: lane l addresses K row l / 4 of
            // them, M offset 4 (l % 4); a step's K rows differ from step 0's by multiples of 4, so their slots agree
            const int k = 8 * (lane / 32) + (lane % 16) / 4;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int granule = (first + 32 * i) / 8 + 2 * ((lane / 16) % 2) + (lane % 4) / 2;
                at[i] = k * Rows + granule_slot<Rows>(k, granule) * 8 + 4 * (lane % 2);
            }
        } else {
            // blocks lie 32 rows apart, which leaves a chunk's slot as it is
            const int row = first + lane % 32;
#pragma unroll
            for (int s = 0; s < kDepth / 16; ++s) at[s] = row * kDepth + chunk_slot(lane % 32, 2 * s + lane / 32) * 8;
        }
    }
    __device__ __forceinline__ void read(const unsigned short* stage, int s, typename T::Fragment (&f)[N]) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr (MN) {
                typedef short s16x4 __attribute__((ext_vector_type(4)));
                const unsigned short* p = stage + at[i] + 16 * s * Rows;
                const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
                const s16x4 hi =
                    __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p + 4 * Rows));
                f[i] = __builtin_bit_cast(typename T::Fragment, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
            } else {
                f[i] = *reinterpret_cast<const typename T::Fragment*>(stage + at[s] + 32 * i * kDepth);
            }
        }
    }
};

// Workgroup b of a product's `total` -> tile: consecutive tiles share operand panels, and each XCD (workgroups go to the 8
// of them in turn) takes a contiguous run of tiles, walked in groups of 4 M tiles.
__device__ __forceinline__ void tile_of(int b, int total, int tiles_m, int tiles_n, int& tm, int& tn, int& split) {
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

// bf16 elements of a stage
template <int TM, int TN>
constexpr int stage_size() {
    return (TM + TN) * kDepth;
}

// Tile `block` of the product's `blocks` by a workgroup of WavesM x WavesN waves; Again: then the tiles `stride` further
// on, of which the first K tile arrives under the epilogue (K must be an even number of K tiles where there are any).
// stage0, stage1: two LDS objects of stage_size (the compiler then tells reads of one from the DMA into the other).
template <typename T, bool AMN, bool BMN, int TM, int TN, int WavesM, int WavesN, int Out, int Kind, bool Again>
__device__ __forceinline__ void make_tiles(const Product& p, int tiles_m, int tiles_n, int block, int blocks, int stride,
                                           unsigned short* stage0, unsigned short* stage1) {
    constexpr int kWaves = WavesM * WavesN;
    constexpr int kThreadCount = kWaves * kWave;
    constexpr int MI = TM / WavesM / 32, NJ = TN / WavesN / 32;
    constexpr bool kGated = Out != kPlain;
    static_assert(!kGated || (!AMN && !BMN && NJ == 2), "a wave's two column blocks are the gate's and the up's");
    constexpr int kOutN = kGated ? TN / 2 : TN;  // output columns of a tile
    constexpr int kStage = stage_size<TM, TN>();
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    const int lane = static_cast<int>(threadIdx.x) % kWave;
    const int wm = wave / WavesN, wn = wave % WavesN;
    int tm, tn, split;
    tile_of(block, blocks, tiles_m, tiles_n, tm, tn, split);
    int m0 = tm * TM, n0 = tn * kOutN;
    bool more = Again && block + stride < blocks;

    Loader<AMN, TM, kWaves> la;
    Loader<BMN, TN, kWaves> lb;
    la.init(p.lda, wave, lane, false);
    lb.init(p.ldb, wave, lane, kGated);

    const int per_segment = (p.k + kDepth - 1) / kDepth;
    const int first_tile = split * p.tiles_per_split;
    const int last_tile = min(first_tile + p.tiles_per_split, per_segment * p.segments);
    int segment = first_tile / per_segment, k0 = (first_tile % per_segment) * kDepth;
    int next_m = m0, next_n = n0;  // the tile that is fetched
    const auto fetch = [&](unsigned short* stage) {
        const int depth = min(kDepth, p.k - k0);
        const int rows_a = min(TM, p.m - next_m), rows_b = min(kOutN, p.n - next_n);
        const unsigned short* a = p.a + segment * p.seg_a + (AMN ? k0 * p.lda + next_m : next_m * p.lda + k0);
        const unsigned short* b = p.b + segment * p.seg_b + (BMN ? k0 * p.ldb + next_n : next_n * p.ldb + k0);
        // M/N-contiguous rows may be read up to their next multiple of 8, which the pitch covers
        la.fetch(a, nullptr, p.lda, AMN ? (rows_a + 7) / 8 * 8 : rows_a, depth, stage, wave);
        lb.fetch(b, kGated ? b + p.up : nullptr, p.ldb, BMN ? (rows_b + 7) / 8 * 8 : rows_b, depth,
                 stage + TM * kDepth, wave);
        k0 += kDepth;
        if (k0 < p.k) return;
        k0 = 0;
        if constexpr (!Again) {
            ++segment;
        } else if (more) {
            tile_of(block + stride, blocks, tiles_m, tiles_n, tm, tn, split);
            next_m = tm * TM, next_n = tn * kOutN;
        }
    };

    gemm::f32x16_t acc[MI][NJ];
    Reader<T, AMN, TM, MI> ra;
    Reader<T, BMN, TN, NJ> rb;
    ra.init(wm * (TM / WavesM), lane);
    rb.init(wn * (TN / WavesN), lane);
    // One K tile from `stage`.  Fragments of the next 16-deep step are read under this step's products, those of the next
    // K tile (in `other`) under the last one's: before it every wave's DMA of that tile has landed and every wave holds
    // its last fragments of this one, so that `stage` takes the K tile after the next (from the late waves in the next K
    // tile's first step, where that stage is `other`).
    typename T::Fragment fa[2][MI], fb[2][NJ];
    const auto read = [&](const unsigned short* stage, int s, int slot) {
        ra.read(stage, s, fa[slot]);
        rb.read(stage + TM * kDepth, s, fb[slot]);
    };
    // half of the waves issue their part of a K tile a step later than the others: 8192 x 1024 x 4096 backward 394 -> 382 us
    const bool late = wave >= kWaves / 2;
    const auto multiply = [&](int slot) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j) acc[i][j] = T::mfma(fa[slot][i], fb[slot][j], acc[i][j]);
        __builtin_amdgcn_sched_barrier(0);
    };
    const int tiles = last_tile - first_tile;
    const auto k_tile = [&](int kt, unsigned short* stage, const unsigned short* other) {
        constexpr int kSteps = kDepth / 16;
        static_assert(kSteps % 2 == 0, "a K tile ends with the second fragments");
#pragma unroll
        for (int s = 0; s + 1 < kSteps; ++s) {
            read(stage, s + 1, (s + 1) % 2);
            if (s == 0 && late && kt >= 1 && (more || kt + 1 < tiles)) fetch(const_cast<unsigned short*>(other));
            multiply(s % 2);
        }
        if (kt + 1 < tiles) {
            stage_barrier();
            if (!late && (more || kt + 2 < tiles)) fetch(stage);
            read(other, 0, 0);
        }
        multiply((kSteps - 1) % 2);
    };
    fetch(stage0);
    stage_barrier();
    for (;;) {
        if (tiles > 1) fetch(stage1);
        read(stage0, 0, 0);
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.0f;
        int kt = 0;
        for (; kt + 1 < tiles; kt += 2) {
            k_tile(kt, stage0, stage1);
            k_tile(kt + 1, stage1, stage0);
        }
        if (kt < tiles) k_tile(kt, stage0, stage1);

        // accumulator element v of lane l: column l % 32, row 8 (v / 4) + 4 (l / 32) + v % 4 of its 32 x 32 block
        const int col = lane % 32, row4 = 4 * (lane / 32);
        if constexpr (!kGated) {
            if (p.d32) {
                const bool direct = p.splits == 1;
                float* d = p.d32 + (direct ? 0 : static_cast<long long>(split) * p.m * p.n);
                const long long ldd = direct ? p.ldd : p.n;
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int j = 0; j < NJ; ++j) {
                        const int c = n0 + wn * (TN / WavesN) + 32 * j + col;
                        if (c >= p.n) continue;
#pragma unroll
                        for (int v = 0; v < 16; ++v) {
                            const int r = m0 + wm * (TM / WavesM) + 32 * i + 8 * (v / 4) + row4 + v % 4;
                            const long long to = direct ? folded(r, p.fold, p.fold_to) : r;
                            if (r < p.m && to >= 0) d[to * ldd + c] = acc[i][j][v];
                        }
                    }
                return;
            }
        }

        // 16-bit outputs leave through LDS, whole tile rows at a time: in MI passes of 32 rows from each row of waves
        constexpr int kPitch = kOutN + 8;
        constexpr int kPassRows = 32 * WavesM;
        static_assert((Out == kBackward ? 2 : 1) * kPassRows * kPitch <= kStage, "a pass fits a stage");
        constexpr int kChunks = kOutN / 8;  // 16-byte pieces of a tile row
        // rows of `out`, whose first `columns` values exist, from LDS
        const auto leave = [&](const unsigned short* lds, unsigned short* out, long long ld, int columns, int pass) {
            const bool wide = reinterpret_cast<std::uintptr_t>(out) % 16 == 0 && ld % 8 == 0;
            for (int q = static_cast<int>(threadIdx.x); q < kPassRows * kChunks; q += kThreadCount) {
                const int local = q / kChunks, c = n0 + q % kChunks * 8;
                const int r = m0 + local / 32 * (TM / WavesM) + 32 * pass + local % 32;
                const long long row = kGated ? r : folded(r, p.fold, p.fold_to);
                if (r >= p.m || row < 0 || c >= columns) continue;
                const unsigned short* in = lds + local * kPitch + q % kChunks * 8;
                unsigned short* to = out + row * ld + c;
                if (wide && c + 8 <= columns) {
                    *reinterpret_cast<u32x4*>(to) = *reinterpret_cast<const u32x4*>(in);
                } else {
                    for (int e = 0; e < 8 && c + e < columns; ++e) to[e] = in[e];
                }
            }
        };
        // backward: this thread's pieces of dh, all of them before the first pass waits for one
        constexpr int kPieces = (kPassRows * kChunks + kThreadCount - 1) / kThreadCount;
        static_assert(kPassRows * kChunks % kThreadCount == 0, "whole pieces");
        u32x4 dh_pieces[Out == kBackward ? MI : 1][kPieces];
        if constexpr (Out == kBackward) {
            const bool wide = reinterpret_cast<std::uintptr_t>(p.dh) % 16 == 0 && p.ld_dh % 8 == 0;
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int k = 0; k < kPieces; ++k) {
                    const int q = static_cast<int>(threadIdx.x) + k * kThreadCount;
                    const int local = q / kChunks, c = n0 + q % kChunks * 8;
                    const int r = m0 + local / 32 * (TM / WavesM) + 32 * i + local % 32;
                    u32x4 piece{0u, 0u, 0u, 0u};
                    if (r < p.m && c < p.n) {
                        const unsigned short* from = p.dh + r * p.ld_dh + c;
                        if (wide && c + 8 <= p.n) {
                            piece = *reinterpret_cast<const u32x4*>(from);
                        } else {
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                if (c + e < p.n) piece[e / 2] |= static_cast<unsigned>(from[e]) << (16 * (e % 2));
                        }
                    }
                    dh_pieces[i][k] = piece;
                }
        }
        unsigned short *one = stage1, *two = stage1 + kPassRows * kPitch;  // stage0 may be taking the next tile
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            lds_barrier();  // the stage is free, and the pass before has left
            if constexpr (Out == kBackward) {
#pragma unroll
                for (int k = 0; k < kPieces; ++k) {
                    const int q = static_cast<int>(threadIdx.x) + k * kThreadCount;
                    *reinterpret_cast<u32x4*>(one + q / kChunks * kPitch + q % kChunks * 8) = dh_pieces[i][k];
                }
                lds_barrier();
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
                    activate<Kind>(acc[i][0][v], value, slope);
                    if constexpr (Out == kForward) {
                        *lds_one = T::rounded(value * up);
                    } else {
                        const float dh = T::value(*lds_one);  // 0 past the last column, and so is what leaves for it
                        *lds_one = T::rounded(dh * up * slope);
                        two[lds_one - one] = T::rounded(dh * value);
                    }
                }
            }
            // the first K tile of the next one has landed: the barrier before the first store, which would be waited for too
            if (Again && i == 0) stage_barrier();
            else lds_barrier();
            if constexpr (Out == kPlain) {
                leave(one, p.d, p.ldd, p.n, i);
            } else if constexpr (Out == kForward) {
                leave(one, p.h, p.ld_h, p.n, i);
            } else {
                leave(one, p.dpre, 2 * p.pitch, static_cast<int>(p.pitch), i);
                leave(two, p.dpre + p.pitch, 2 * p.pitch, static_cast<int>(p.pitch), i);
            }
        }
        if (!more) return;
        lds_barrier();  // stage1 is free
        block += stride;
        m0 = next_m, n0 = next_n;
        more = block + stride < blocks;
    }
}

// The waves of a tile of `Edge` rows and columns: 256 takes 2 x 4 of 128 x 64 outputs, 128 2 x 2 of 64 x 64, 64 2 x 1 of 32 x 64.
template <int Edge>
struct Waves {
    static constexpr int kM = 2, kN = Edge == 256 ? 4 : Edge == 128 ? 2 : 1;
    static constexpr int kThreads = kM * kN * kWave;
};

// Whether a workgroup goes on to other tiles: 8192 x 512 -> 2048 43 -> 40.5 us, 16384 x 2048 -> 8192 910 -> 887 us; the
// backward projection, whose epilogue waits for its own loads, gains nothing.
template <int Edge, int Out>
__host__ __device__ constexpr bool tiles_follow() {
    return Edge == 256 && Out == kForward;
}

template <typename T, int Edge, int Out, int Kind>
__global__ __launch_bounds__(Waves<Edge>::kThreads, 1) void project_kernel(Product p, int tiles_m, int tiles_n) {
    __shared__ __attribute__((aligned(1024))) unsigned short stage0[stage_size<Edge, Edge>()];
    __shared__ __attribute__((aligned(1024))) unsigned short stage1[stage_size<Edge, Edge>()];
    make_tiles<T, false, false, Edge, Edge, Waves<Edge>::kM, Waves<Edge>::kN, Out, Kind, tiles_follow<Edge, Out>()>(
        p, tiles_m, tiles_n, static_cast<int>(blockIdx.x), tiles_m * tiles_n, static_cast<int>(gridDim.x), stage0, stage1);
}

// One of the two gradient products: its tiles, and its workgroups (0: not asked for).
struct Share {
    Product p;
    int tiles_m, tiles_n, blocks;
};

// dx and dW side by side in one launch, the workgroups with more of K first: together they fill the CUs where each alone
// would not (8192 x 1024 x 4096: 128 tiles of 256 x 256 each; 255 us together, 2 x 148 us one after the other on tiles of
// 128 x 128).
template <typename T, int Edge>
__global__ __launch_bounds__(Waves<Edge>::kThreads, 1) void gradients_kernel(Share dx, Share dw, int dw_first) {
    __shared__ __attribute__((aligned(1024))) unsigned short stage0[stage_size<Edge, Edge>()];
    __shared__ __attribute__((aligned(1024))) unsigned short stage1[stage_size<Edge, Edge>()];
    const int block = static_cast<int>(blockIdx.x);
    if (dw_first ? block >= dw.blocks : block < dx.blocks)
        make_tiles<T, false, true, Edge, Edge, Waves<Edge>::kM, Waves<Edge>::kN, kPlain, kRelu, false>(
            dx.p, dx.tiles_m, dx.tiles_n, dw_first ? block - dw.blocks : block, dx.blocks, 0, stage0, stage1);
    else
        make_tiles<T, true, true, Edge, Edge, Waves<Edge>::kM, Waves<Edge>::kN, kPlain, kRelu, false>(
            dw.p, dw.tiles_m, dw.tiles_n, dw_first ? block : block - dx.blocks, dw.blocks, 0, stage0, stage1);
}

// What a tile takes: up to `beside` workgroups a CU, r of them on each; us per 64 of K and us beside that.  Measured with
// bf16 over K = 1024 on tiles of 256 / 128 / 64: 8192 x 4096 outputs 140 / 154 / 239 us, 1024 x 4096 31 / 22.5 / 33 us, 256 x
// 4096 28 / 13.5 / 12.9 us.
struct TileCost {
    int edge, beside;
    double step, fixed, fixed_beside;
    // 0.6 us at least a step: the loads' latency
    double time(double steps, double r) const { return steps * std::max(step * r, 0.6) + fixed + fixed_beside * r; }
};
constexpr TileCost kTileCosts[] = {{256, 1, 1.8, 5.0, 0.0}, {128, 2, 0.5, 1.5, 0.7}, {64, 5, 0.23, 1.0, 0.3}};
constexpr int kCus = 256;

inline long long tiles_of(long long m, long long n, int edge) {
    return static_cast<long long>(ceil_div(m, edge)) * ceil_div(n, edge);
}

// The tile that projects m rows onto n columns (gate and up) over k_tiles 64ths of K soonest.
int projection_tile(long long m, long long n, long long k_tiles) {
    int best = 64;
    double least = 1e30;
    for (const TileCost& c : kTileCosts) {
        const long long tiles = tiles_of(m, n, c.edge), slots = kCus * c.beside, rest = tiles % slots;
        const double steps = static_cast<double>(k_tiles);
        const double time = static_cast<double>(tiles / slots) * c.time(steps, c.beside) +
                            (rest ? c.time(steps, static_cast<double>(ceil_div(rest, kCus))) : 0.0);
        if (time < least) {
            least = time;
            best = c.edge;
        }
    }
    return best;
}

// The tile of both gradient products and the K splits of each (whose fp32 sums cost a launch and their bytes).  It goes
// by the sizes alone: one gradient has the same bits whether the other is asked for or not.
struct GradientPlan {
    int edge, dx_splits, dw_splits;
};
constexpr int kMostSplits = 64;

GradientPlan gradient_plan(long long dx_m, long long dw_m, long long n, long long dx_tiles, long long dw_tiles) {
    GradientPlan best{64, 1, 1};
    double least = 1e30;
    for (const TileCost& c : kTileCosts) {
        const long long dx_groups = tiles_of(dx_m, n, c.edge), dw_groups = tiles_of(dw_m, n, c.edge), slots = kCus * c.beside;
        for (int a = 1; a <= kMostSplits && (a == 1 || dx_tiles / a >= 4); a *= 2) {
            for (int b = 1; b <= kMostSplits && (b == 1 || dw_tiles / b >= 4); b *= 2) {
                const long long groups = dx_groups * a + dw_groups * b;
                const double r = groups <= slots ? static_cast<double>(ceil_div(groups, kCus)) : c.beside;
                const double dx = c.time(static_cast<double>(ceil_div(dx_tiles, a)), r);
                const double dw = c.time(static_cast<double>(ceil_div(dw_tiles, b)), r);
                double time = std::max(dx, dw);
                if (groups > slots) time = 0.5 * time + (dx * dx_groups * a + dw * dw_groups * b) / slots;
                if (a > 1 || b > 1)
                    time += 4.0 + ((a > 1 ? a * dx_m : 0) + (b > 1 ? b * dw_m : 0)) * static_cast<double>(n) * 8.0 / 4.5e6;
                if (time < least) {
                    least = time;
                    best = {c.edge, a, b};
                }
                if (groups > 4 * slots) break;
            }
        }
    }
    return best;
}

template <typename T, int Edge, int Out, int Kind>
void launch_projection(const Product& p, hipStream_t stream) {
    const long long tiles_m = ceil_div(p.m, Edge), tiles_n = ceil_div(p.n, Edge / 2);
    // an even number of K tiles: each CU's workgroup takes its tiles one after the other
    const bool again = tiles_follow<Edge, Out>() && ceil_div(p.k, kDepth) % 2 == 0;
    const long long groups = again ? std::min<long long>(tiles_m * tiles_n, kCus) : tiles_m * tiles_n;
    hipLaunchKernelGGL((project_kernel<T, Edge, Out, Kind>), dim3(static_cast<unsigned>(groups)),
                       dim3(Waves<Edge>::kThreads), 0, stream, p, static_cast<int>(tiles_m), static_cast<int>(tiles_n));
    check_launch("Launch gated projection");
}

template <typename T, int Out, int Kind>
void launch_projection(const Product& p, int edge, hipStream_t stream) {
    if (edge == 256) launch_projection<T, 256, Out, Kind>(p, stream);
    else if (edge == 128) launch_projection<T, 128, Out, Kind>(p, stream);
    else launch_projection<T, 64, Out, Kind>(p, stream);
}

// ---------------------------------------------------------------------------
// Few rows: the weights stream through the matrix cores once
// ---------------------------------------------------------------------------
// A workgroup makes 16 hidden values of up to 16 Tiles rows of x: its 4 waves take turns over K, 64 values a step, whose
// pieces each lane loads straight into the fragments of v_mfma_f32_16x16x32 (lane l: weight row, or row of x, l % 16,
// and K 16 (l / 16) .. + 15 of the step, so that a row's 128 bytes are read by two instructions), and the waves' sums
// meet in LDS.  No staging, and no barrier before the end; rows of any alignment.  Bound by the weights' stream: one row over
// 2 x 4096 x 1024 bf16 5.1 us (3.3 TB/s, the launch included), over 2 x 16384 x 4096 57 us (4.7 TB/s).  64 rows x 512 x 2048
// fp16 6.2 us, on tiles of 64 7.0 us; past 64 rows the tiles are the faster ones.
constexpr int kStreamRows = 64;  // most rows

struct __attribute__((packed, aligned(2))) Piece {
    unsigned w[4];
};

// Eight values of a row from k on; Whole: all inside the row, else zeros past its end.
template <typename T, bool Whole>
__device__ __forceinline__ typename T::Fragment row_piece(const unsigned short* row, int k, int columns) {
    if (Whole || k + 8 <= columns) {
        const Piece piece = *reinterpret_cast<const Piece*>(row + k);
        return __builtin_bit_cast(typename T::Fragment, piece);
    }
    Piece piece{};
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (k + e < columns) piece.w[e / 2] |= static_cast<unsigned>(row[k + e]) << (16 * (e % 2));
    return __builtin_bit_cast(typename T::Fragment, piece);
}

template <typename T, int Tiles, int Out, int Kind>
__global__ __launch_bounds__(256) void stream_kernel(Product p) {
    constexpr int kWaves = 4;
    __shared__ f32x4 sums[kWaves][Tiles][2][kWave];
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    const int lane = static_cast<int>(threadIdx.x) % kWave;
    const int n0 = static_cast<int>(blockIdx.x) * 16;
    // rows past the end repeat the last: what they make is not written
    const unsigned short* gate = p.b + min(n0 + lane % 16, p.n - 1) * p.ldb;
    const unsigned short* up = gate + p.up;
    const unsigned short* x[Tiles];
#pragma unroll
    for (int i = 0; i < Tiles; ++i) x[i] = p.a + min(16 * i + lane % 16, p.m - 1) * p.lda;
    f32x4 acc[Tiles][2];
#pragma unroll
    for (int i = 0; i < Tiles; ++i) acc[i][0] = acc[i][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const auto step = [&](int k0, auto whole) {
        constexpr bool kWhole = decltype(whole)::value;
        const int k = k0 + 16 * (lane / 16);
        typename T::Fragment g[2], u[2], rows[Tiles][2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            g[s] = row_piece<T, kWhole>(gate, k + 8 * s, p.k);
            u[s] = row_piece<T, kWhole>(up, k + 8 * s, p.k);
#pragma unroll
            for (int i = 0; i < Tiles; ++i) rows[i][s] = row_piece<T, kWhole>(x[i], k + 8 * s, p.k);
        }
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < Tiles; ++i) {
                acc[i][0] = T::mfma16(g[s], rows[i][s], acc[i][0]);
                acc[i][1] = T::mfma16(u[s], rows[i][s], acc[i][1]);
            }
    };
    int k0 = 64 * wave;
    constexpr int kTurn = 64 * kWaves;
    for (; k0 + 3 * kTurn + 64 <= p.k; k0 += 4 * kTurn) {
#pragma unroll
        for (int turn = 0; turn < 4; ++turn) step(k0 + turn * kTurn, std::true_type{});
    }
    for (; k0 + 64 <= p.k; k0 += kTurn) step(k0, std::true_type{});
    if (k0 < p.k) step(k0, std::false_type{});
#pragma unroll
    for (int i = 0; i < Tiles; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) sums[wave][i][h][lane] = acc[i][h];
    __syncthreads();
    // wave i finishes rows 16 i ..: lane l holds row l % 16 and hidden values 4 (l / 16) .. + 3
    const int i = wave;
    const int r = 16 * i + lane % 16, c = n0 + 4 * (lane / 16);
    if (i >= Tiles || r >= p.m) return;
    f32x4 z[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        z[h] = sums[0][i][h][lane];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) z[h] += sums[w][i][h][lane];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float value, slope;
        activate<Kind>(z[0][e], value, slope);
        if constexpr (Out == kForward) {
            if (c + e < p.n) p.h[r * p.ld_h + c + e] = T::rounded(value * z[1][e]);
        } else {
            if (c + e >= p.pitch) continue;
            const bool pad = c + e >= p.n;  // zeroed
            const float dh = pad ? 0.0f : T::value(p.dh[r * p.ld_dh + c + e]);
            p.dpre[r * 2 * p.pitch + c + e] = pad ? 0 : T::rounded(dh * z[1][e] * slope);
            p.dpre[r * 2 * p.pitch + p.pitch + c + e] = pad ? 0 : T::rounded(dh * value);
        }
    }
}

template <typename T, int Out, int Kind>
void launch_stream(const Product& p, hipStream_t stream) {
    const dim3 grid(ceil_div(p.n, 16)), block(256);
    if (p.m <= 16) hipLaunchKernelGGL((stream_kernel<T, 1, Out, Kind>), grid, block, 0, stream, p);
    else if (p.m <= 32) hipLaunchKernelGGL((stream_kernel<T, 2, Out, Kind>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((stream_kernel<T, 4, Out, Kind>), grid, block, 0, stream, p);
    check_launch("Launch gated stream");
}

// Copies of operands whose rows the DMA cannot read in 16-byte pieces: to[r, 0 .. pitch) = from[r, 0 .. columns), then zeros.
struct Copy {
    const unsigned short* from;
    unsigned short* to;
    long long ld, rows;
    int columns, pitch;
    __host__ __device__ long long pieces() const { return rows * (pitch / 8); }
};
__global__ __launch_bounds__(256) void pack_kernel(Copy a, Copy b) {
    const long long all = a.pieces() + b.pieces();
    for (long long i = blockIdx.x * 256LL + threadIdx.x; i < all; i += gridDim.x * 256LL) {
        const bool second = i >= a.pieces();
        const Copy& copy = second ? b : a;
        const long long q = second ? i - a.pieces() : i;
        const long long r = q / (copy.pitch / 8);
        const int c = static_cast<int>(q % (copy.pitch / 8)) * 8;
        const unsigned short* s = copy.from + r * copy.ld + c;
        unsigned w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const unsigned lo = c + 2 * e < copy.columns ? s[2 * e] : 0u, hi = c + 2 * e + 1 < copy.columns ? s[2 * e + 1] : 0u;
            w[e] = lo | (hi << 16);
        }
        *reinterpret_cast<u32x4*>(copy.to + r * copy.pitch + c) = u32x4{w[0], w[1], w[2], w[3]};
    }
}

// fp32: gate and up of `pre` [rows, 2 hidden] -> h
template <int Kind>
__global__ __launch_bounds__(256) void gate_forward(const float* pre, float* h, long long ld_h, long long rows, int hidden) {
    const long long n = rows * hidden;
    for (long long q = blockIdx.x * 256LL + threadIdx.x; q < n; q += gridDim.x * 256LL) {
        const long long r = q / hidden, at = 2 * r * hidden + q % hidden;
        float value, slope;
        activate<Kind>(pre[at], value, slope);
        h[r * ld_h + q % hidden] = value * pre[at + hidden];
    }
}

// fp32: gate and up of `pre` become their gradients.
template <int Kind>
__global__ __launch_bounds__(256) void gate_backward(float* pre, const float* dh, long long ld_dh, long long rows,
                                                     int hidden) {
    const long long n = rows * hidden;
    for (long long q = blockIdx.x * 256LL + threadIdx.x; q < n; q += gridDim.x * 256LL) {
        const long long r = q / hidden, at = 2 * r * hidden + q % hidden;
        float value, slope;
        activate<Kind>(pre[at], value, slope);
        const float d = dh[r * ld_dh + q % hidden], up = pre[at + hidden];
        pre[at] = d * up * slope;
        pre[at + hidden] = d * value;
    }
}

// Both products' splits, in their order (splits 1: nothing to add).
struct Sum {
    Product p;
    const float* partial;
    int splits;
    __host__ __device__ long long values() const { return splits > 1 ? static_cast<long long>(p.m) * p.n : 0; }
};
template <typename T>
__global__ __launch_bounds__(256) void reduce_kernel(Sum a, Sum b) {
    const long long all = a.values() + b.values();
    for (long long i = blockIdx.x * 256LL + threadIdx.x; i < all; i += gridDim.x * 256LL) {
        const bool second = i >= a.values();
        const Sum& s = second ? b : a;
        const long long q = second ? i - a.values() : i, total = s.values();
        const long long row = folded(static_cast<int>(q / s.p.n), s.p.fold, s.p.fold_to);
        if (row < 0) continue;
        float sum = 0.0f;
#pragma unroll 4
        for (int k = 0; k < s.splits; ++k) sum += s.partial[k * total + q];
        const long long at = row * s.p.ldd + q % s.p.n;
        if (s.p.d32) s.p.d32[at] = sum;
        else s.p.d[at] = T::rounded(sum);
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

GradientPlan plan_of(const Sizes& s) {
    return gradient_plan(s.rows, 2 * align8(s.hidden), s.inputs, 2LL * ceil_div(s.hidden, kDepth), ceil_div(s.rows, kDepth));
}

struct Layout {
    std::size_t x, w, dpre, dx_sums, dw_sums, bytes;
    GradientPlan plan;
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
        l.plan = plan_of(s);
        l.dx_sums = take(l.plan.dx_splits > 1 ? l.plan.dx_splits * s.rows * s.inputs : 0, 4);
        l.dw_sums = take(l.plan.dw_splits > 1 ? l.plan.dw_splits * 2 * hidden_pitch * s.inputs : 0, 4);
    }
    l.bytes = at;
    return l;
}

// K splits of the fp32 products, as the framework splits its own: the projection's and the input gradient's to 1024 tiles
// of 64 x 64, 256 of K each; the weight gradient's to 512 of 128 x 128, 384 of K each, where that makes 256 of them.
// Shorter sums are more exact, too: 14 x 1768 -> 1720 35 -> 19 us and 1.0e-6 -> 5.1e-7 of the output's norm.
int fp32_splits(long long rows, long long columns, long long k) {
    const long long tiles = static_cast<long long>(ceil_div(rows, 64)) * ceil_div(columns, 64);
    int splits = 1;
    while (tiles * splits < 1024 && k / (2 * splits) >= 256 && splits < 16) splits *= 2;
    return splits;
}
int fp32_pre_splits(const Sizes& s) { return fp32_splits(s.rows, 2LL * s.hidden, s.inputs); }
int fp32_dx_splits(const Sizes& s) { return fp32_splits(s.rows, s.inputs, 2LL * s.hidden); }
int fp32_dw_splits(const Sizes& s) {
    const long long m = 2LL * s.hidden, n = s.inputs;
    int splits = 1;
    if (m > 64 && n > 64) {
        const long long wide = static_cast<long long>(ceil_div(m, 128)) * ceil_div(n, 128);
        while (wide * splits < 512 && splits * 2 <= s.rows / 384 && splits < 256) splits *= 2;
        if (wide * splits >= 256) return splits;
        splits = 1;
    }
    const long long tiles = static_cast<long long>(ceil_div(m, 64)) * ceil_div(n, 64), steps = (s.rows + 15) / 16;
    while (tiles * splits < 1024 && splits * 2 <= std::max<long long>(1, steps / (m * n <= 65536 ? 4 : 16)) && splits < 256)
        splits *= 2;
    return splits;
}

std::size_t fp32_partial_bytes(const Sizes& s, bool backward) {
    const std::size_t pre = rl_gemm_workspace(2, static_cast<int>(s.rows), 2 * s.hidden, s.inputs, 1, fp32_pre_splits(s));
    if (!backward) return pre;
    const std::size_t dx = rl_gemm_workspace(2, static_cast<int>(s.rows), s.inputs, 2 * s.hidden, 1, fp32_dx_splits(s));
    const std::size_t dw = rl_gemm_workspace(2, 2 * s.hidden, s.inputs, static_cast<int>(s.rows), 1, fp32_dw_splits(s));
    return std::max(pre, std::max(dx, dw));
}

std::size_t fp32_bytes(const Sizes& s, bool backward) {
    return aligned_bytes(static_cast<std::size_t>(2 * s.rows * s.hidden) * 4) + fp32_partial_bytes(s, backward);
}

std::size_t workspace_bytes(const Sizes& s, bool backward) {
    if (s.rows == 0) return 0;
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
    const int rows = static_cast<int>(s.rows), in = s.inputs, both = 2 * s.hidden;
    const float *x = static_cast<const float*>(o.x), *w = static_cast<const float*>(o.w);
    float* pre = reinterpret_cast<float*>(o.workspace);  // [rows, 2 hidden]: gate, up
    const long long each = s.rows * s.hidden;
    float* partial = reinterpret_cast<float*>(o.workspace + aligned_bytes(static_cast<std::size_t>(2 * each) * 4));
    const std::size_t bytes = fp32_partial_bytes(s, backward);
    const int pre_splits = fp32_pre_splits(s);
    run_gemm(2, 0, 0, 1, 1, rows, both, in, 1, x, o.ldx, 0, w, in, 0, nullptr, pre, both, 0, nullptr, 0, 0.0f, 0, pre_splits,
             pre_splits > 1 ? partial : nullptr, bytes, stream, nullptr, nullptr, nullptr);
    if (!backward) {
        with_activation(o.activation, [&](auto kind) {
            hipLaunchKernelGGL((gate_forward<decltype(kind)::value>), dim3(blocks_for(each)), dim3(256), 0, stream, pre,
                               static_cast<float*>(o.h), o.ld_h, s.rows, s.hidden);
        });
        check_launch("Launch gating");
        return;
    }
    with_activation(o.activation, [&](auto kind) {
        hipLaunchKernelGGL((gate_backward<decltype(kind)::value>), dim3(blocks_for(each)), dim3(256), 0, stream, pre,
                           static_cast<const float*>(o.dh), o.ld_dh, s.rows, s.hidden);
    });
    check_launch("Launch gating gradient");
    if (o.dx) {
        const int splits = fp32_dx_splits(s);
        run_gemm(2, 0, 0, 1, 0, rows, in, both, 1, pre, both, 0, w, in, 0, nullptr, static_cast<float*>(o.dx), o.ld_dx, 0,
                 nullptr, 0, 0.0f, 0, splits, splits > 1 ? partial : nullptr, bytes, stream, nullptr, nullptr, nullptr);
    }
    if (o.dw) {
        const int splits = fp32_dw_splits(s);
        run_gemm(2, 0, 0, 0, 0, both, in, rows, 1, pre, both, 0, x, o.ldx, 0, nullptr, static_cast<float*>(o.dw), in, 0,
                 nullptr, 0, 0.0f, 0, splits, splits > 1 ? partial : nullptr, bytes, stream, nullptr, nullptr, nullptr);
    }
}

// A gradient product's share of the launch: `splits` pieces of K, whose sums go to `sums` where they are several.
Share share_of(const Product& p, int edge, int splits, float* sums) {
    Share share{p, static_cast<int>(ceil_div(p.m, edge)), static_cast<int>(ceil_div(p.n, edge)), 0};
    const int tiles = static_cast<int>(ceil_div(p.k, kDepth)) * p.segments;
    share.p.tiles_per_split = static_cast<int>(ceil_div(tiles, splits));
    share.p.splits = static_cast<int>(ceil_div(tiles, share.p.tiles_per_split));
    const long long blocks = static_cast<long long>(share.tiles_m) * share.tiles_n * share.p.splits;
    require(blocks <= INT_MAX / 2, "The gated product has too many tiles.");
    share.blocks = static_cast<int>(blocks);
    if (share.p.splits > 1) {
        share.p.d = nullptr;
        share.p.d32 = sums;
    }
    return share;
}

template <typename T, int Edge>
void launch_gradients(const Share& dx, const Share& dw, hipStream_t stream) {
    const int dw_first = dw.p.tiles_per_split > dx.p.tiles_per_split;
    hipLaunchKernelGGL((gradients_kernel<T, Edge>), dim3(static_cast<unsigned>(dx.blocks + dw.blocks)),
                       dim3(Waves<Edge>::kThreads), 0, stream, dx, dw, dw_first);
    check_launch("Launch gated gradients");
}

// The operand as the DMA reads it: in place, or (`copy` filled in) in a copy with rows of 16-byte pieces.
const unsigned short* readable(const void* data, long long rows, int columns, long long& ld, char* space, Copy& copy) {
    const unsigned short* p = static_cast<const unsigned short*>(data);
    if (aligned(p, 16) && columns % 8 == 0 && (ld % 8 == 0 || rows == 1) && ld <= kMaxPitch) {
        if (rows == 1) ld = align8(columns);
        return p;
    }
    unsigned short* to = reinterpret_cast<unsigned short*>(space);
    copy = Copy{p, to, ld, rows, columns, static_cast<int>(align8(columns))};
    ld = copy.pitch;
    return to;
}

template <typename T>
void run_16bit(const Sizes& s, const Operands& o, const Layout& l, bool backward, hipStream_t stream) {
    const bool few = s.rows <= kStreamRows;
    long long ldx = o.ldx, ldw = s.inputs;
    const unsigned short *x = static_cast<const unsigned short*>(o.x), *w = static_cast<const unsigned short*>(o.w);
    if (!few || backward) {
        Copy copies[2]{};
        copies[0].pitch = copies[1].pitch = 8;
        x = readable(o.x, s.rows, s.inputs, ldx, o.workspace + l.x, copies[0]);
        w = readable(o.w, 2LL * s.hidden, s.inputs, ldw, o.workspace + l.w, copies[1]);
        const long long pieces = copies[0].pieces() + copies[1].pieces();
        if (pieces > 0) {
            hipLaunchKernelGGL(pack_kernel, dim3(blocks_for(pieces)), dim3(256), 0, stream, copies[0], copies[1]);
            check_launch("Launch operand copies");
        }
    }
    Product p{};
    p.a = x;
    p.lda = ldx;
    p.b = w;
    p.ldb = ldw;
    p.up = s.hidden * ldw;
    p.m = static_cast<int>(s.rows);
    p.n = s.hidden;
    p.k = few ? s.inputs : static_cast<int>(align8(s.inputs));
    p.segments = 1;
    p.splits = 1;
    p.tiles_per_split = static_cast<int>(ceil_div(p.k, kDepth));
    p.h = static_cast<unsigned short*>(o.h);
    p.ld_h = o.ld_h;
    const int edge = projection_tile(s.rows, 2LL * s.hidden, p.tiles_per_split);
    const auto project = [&](auto out) {
        with_activation(o.activation, [&](auto kind) {
            constexpr int kOut = decltype(out)::value, kKind = decltype(kind)::value;
            if (few) launch_stream<T, kOut, kKind>(p, stream);
            else launch_projection<T, kOut, kKind>(p, edge, stream);
        });
    };
    if (!backward) {
        project(std::integral_constant<int, kForward>{});
        return;
    }
    const long long pitch = align8(s.hidden);
    unsigned short* dpre = reinterpret_cast<unsigned short*>(o.workspace + l.dpre);
    p.dh = static_cast<const unsigned short*>(o.dh);
    p.ld_dh = o.ld_dh;
    p.dpre = dpre;
    p.pitch = pitch;
    project(std::integral_constant<int, kBackward>{});

    const GradientPlan& plan = l.plan;
    Product dx{}, dw{};
    dx.a = dw.a = dpre;
    dx.lda = dw.lda = 2 * pitch;
    dx.n = dw.n = s.inputs;
    dx.m = static_cast<int>(s.rows);
    dx.k = s.hidden;
    dx.segments = 2;
    dx.seg_a = pitch;
    dx.b = w;
    dx.ldb = ldw;
    dx.seg_b = s.hidden * ldw;
    dx.fold = dx.fold_to = INT_MAX;
    dx.d = static_cast<unsigned short*>(o.dx);
    dx.ldd = o.ld_dx;
    dw.m = static_cast<int>(2 * pitch);
    dw.k = static_cast<int>(s.rows);
    dw.segments = 1;
    dw.b = x;
    dw.ldb = ldx;
    dw.fold = static_cast<int>(pitch);
    dw.fold_to = s.hidden;
    if (o.dw_fp32) dw.d32 = static_cast<float*>(o.dw);
    else dw.d = static_cast<unsigned short*>(o.dw);
    dw.ldd = s.inputs;
    float *dx_sums = reinterpret_cast<float*>(o.workspace + l.dx_sums), *dw_sums = reinterpret_cast<float*>(o.workspace + l.dw_sums);
    Share dx_share = share_of(dx, plan.edge, plan.dx_splits, dx_sums), dw_share = share_of(dw, plan.edge, plan.dw_splits, dw_sums);
    if (!o.dx) dx_share.blocks = 0;
    if (!o.dw) dw_share.blocks = 0;
    if (plan.edge == 256) launch_gradients<T, 256>(dx_share, dw_share, stream);
    else if (plan.edge == 128) launch_gradients<T, 128>(dx_share, dw_share, stream);
    else launch_gradients<T, 64>(dx_share, dw_share, stream);
    const Sum dx_sum{dx, dx_sums, o.dx ? dx_share.p.splits : 0}, dw_sum{dw, dw_sums, o.dw ? dw_share.p.splits : 0};
    const long long values = dx_sum.values() + dw_sum.values();
    if (values > 0) {
        hipLaunchKernelGGL((reduce_kernel<T>), dim3(blocks_for(values)), dim3(256), 0, stream, dx_sum, dw_sum);
        check_launch("Launch gated gradient sums");
    }
}

struct Span {
    const void* begin;
    std::size_t bytes;
    bool meets(const Span& o) const {
        const char *a = static_cast<const char*>(begin), *b = static_cast<const char*>(o.begin);
        return a && b && bytes && o.bytes && a < b + o.bytes && b < a + bytes;
    }
};

void check_sizes(const Sizes& s) {
    require(s.type == 0 || s.type == 1 || s.type == 3, "Gated products take operands of type 0 (fp32), 1 (bf16) or 3 (fp16).");
    require(s.rows >= 0 && s.rows <= (1 << 24) && s.inputs > 0 && s.hidden > 0 && s.inputs <= (1 << 20) &&
                s.hidden <= (1 << 20),
            "Gated products take 0 to 2^24 rows and 1 to 2^20 inputs and hidden values.");
    require(2LL * s.inputs * s.hidden <= INT_MAX && 2 * s.rows * s.hidden <= INT_MAX &&
                s.rows * s.inputs <= INT_MAX,
            "A gated product's matrices (both halves of them) hold at most 2^31 - 1 values each.");
}

void run(const Sizes& s, const Operands& o, std::size_t bytes, bool backward, hipStream_t stream) {
    check_sizes(s);
    require(o.activation >= kSilu && o.activation <= kRelu, "Unknown activation: 0 silu, 1 gelu, 2 relu.");
    Layout layout{};
    if (s.rows > 0 && s.type != 0) layout = layout_of(s, backward);
    const std::size_t need = s.rows == 0 ? 0 : s.type == 0 ? fp32_bytes(s, backward) : layout.bytes;
    require(need == 0 || (o.workspace && bytes >= need && aligned(o.workspace, 16)),
            "The gated workspace is null, misaligned or too small (rl_gated_workspace).");
    const int size = s.type == 0 ? 4 : 2;
    for (const void* q : {o.x, o.w, o.dh, static_cast<const void*>(o.h), static_cast<const void*>(o.dx)})
        require(aligned(q, size), "Gated operands must be aligned to their elements.");
    require(aligned(o.dw, o.dw_fp32 ? 4 : size), "Gated operands must be aligned to their elements.");
    require(s.rows <= 1 || (o.ldx >= s.inputs && (!o.h || o.ld_h >= s.hidden) && (!o.dh || o.ld_dh >= s.hidden) &&
                            (!o.dx || o.ld_dx >= s.inputs)),
            "The rows of a gated operand overlap.");
    // what is written lies apart from what is read
    const std::size_t weights = 2 * static_cast<std::size_t>(s.hidden) * s.inputs;
    const auto bytes_of = [&](long long ld, int columns, int each) {
        return s.rows ? (static_cast<std::size_t>(s.rows - 1) * (s.rows > 1 ? ld : 0) + columns) * each : 0;
    };
    const Span read[] = {{o.x, bytes_of(o.ldx, s.inputs, size)}, {o.w, weights * size}, {o.dh, bytes_of(o.ld_dh, s.hidden, size)}};
    const Span written[] = {{o.h, bytes_of(o.ld_h, s.hidden, size)},
                            {o.dx, bytes_of(o.ld_dx, s.inputs, size)},
                            {o.dw, weights * (o.dw_fp32 ? 4 : size)},
                            {o.workspace, need}};
    for (const Span& out : written) {
        for (const Span& in : read) require(!out.meets(in), "An output or the workspace of a gated product overlaps an input.");
        for (const Span& other : written)
            require(&other == &out || !out.meets(other), "Outputs and workspace of a gated product overlap.");
    }
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
    else if (s.type == 1) run_16bit<Bf16>(s, o, layout, backward, stream);
    else run_16bit<F16>(s, o, layout, backward, stream);
}

}  // namespace gated
}  // namespace rl

RL_API size_t rl_gated_workspace(int type, long long rows, int inputs, int hidden, int backward) {
    std::size_t bytes = 0;
    rl::guarded("rl_gated_workspace", [&] {
        const rl::gated::Sizes s{type, rows, inputs, hidden};
        rl::gated::check_sizes(s);
        bytes = rl::gated::workspace_bytes(s, backward != 0);
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
