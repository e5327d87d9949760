// Matrix products of the cross entropy of a linear head (ds_vocab*.hip): one tiled kernel, whose operands may lie either way
// and whose results go through the epilogue of the step that they belong to.
//
//   logits     s[t][v] = sum_d W[v][d] h[t][d] + b[v]        both operands contiguous along the reduction
//   dhidden    dh[t][d] = sum_v W[v][d] P[t][v]              W contiguous across it
//   dweight    dW[v][d] = sum_t h[t][d] P[t][v]              both contiguous across it
//
// Every product is C[n][m] = sum_k A(m, k) B(n, k): a lane of the matrix instruction holds four neighbouring m of one n, so
// results are written along m, and what is summed over the vocabulary (m of the logits) is summed inside a lane first.
//
// float32 operands come as three bfloat16 planes, x = x0 + 2^-8 x1 + 2^-16 x2, and a product is the sum of the six plane
// products above 2^-24 of it (x0 y0, x0 y1, x1 y0, x1 y1, x0 y2, x2 y0): six times the bf16 work at a rate of bf16, where the
// float32 matrix instructions take sixteen times the time of bf16.  The planes' factors keep all 24 bits of the smallest
// values, which planes without them would lose below 2^-110.  Results that infinities make NaN in them are formed again from
// the largest planes (product_tile).
//
// What bounds them: large ones the power of the chip, which holds the clock at 1.5 to 1.6 GHz while the matrix cores are busy 70
// to 85 % of the cycles (a library's products of the same sizes run at the same rate).  A piece of 8192 tokens x 65536 words x
// 4096 features, bfloat16, 4.4 TFLOP each: scores 3.2 ms, with their exponentials 3.7 ms, probabilities 3.5 ms, hidden gradients
// 3.15 ms, weight gradients 3.2 ms, 1.2 to 1.4 PFLOP/s; plain library products of these operands take 3.24, 3.43 and 3.92 ms.  float32, 2048 tokens x 32768 words x
// 1024 features, 137 GFLOP each: 0.68 to 0.85 ms, 1.0 to 1.2 PFLOP/s of plane products, 160 to 200 TFLOP/s of float32, where the
// library reaches 154.  Few tokens are bound by reading the weights (37 tokens, 50021 words x 2048, bfloat16: 205 MB in 41 us),
// small problems by what one CU can fetch at a time, some 50 bytes per ns from other XCDs' results: hence the small tiles.
#pragma once
#include "ds_train.h"
#include <type_traits>

namespace ds {
namespace vocab {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// The 16-bit type that the matrix instructions take, and how many planes of it make a value.
// `step` is the reduction of a stage: rows of 128 bytes, a cache line, for operands along k.  (Half of it, with twice the
// stages, fetched every line twice.)  float32's planes lie 64 bytes of each after the other, and make up 192.
struct Bf16 { static constexpr int planes = 1, step = 64, unit = 32; static constexpr bool half = false; };
struct F16 { static constexpr int planes = 1, step = 64, unit = 32; static constexpr bool half = true; };
struct Split { static constexpr int planes = 3, step = 32, unit = 16; static constexpr bool half = false; };  // float32

// A matrix instruction: unit x unit results, 16 x 16 from 32 of the reduction or 32 x 32 from 16.  Lane l has one n,
// l % unit, and `groups` times four neighbouring m.
template <typename P>
struct Unit {
    static constexpr int size = P::unit, groups = size == 32 ? 4 : 1, depth = size == 32 ? 16 : 32;
    typedef typename std::conditional<size == 32, f32x16, f32x4>::type Result;

    template <typename V> __device__ static __forceinline__ V as(s16x8 v) { return __builtin_bit_cast(V, v); }

    // first m of a lane, and of its groups behind that
    __device__ static __forceinline__ int lane_m(int lane) { return lane / size * 4; }
    static constexpr int group_m(int q) { return q * 8; }

    __device__ static __forceinline__ Result multiply(s16x8 a, s16x8 b, Result c)
    {
        if constexpr (size == 32) {
            if constexpr (P::half)
                return __builtin_amdgcn_mfma_f32_32x32x16_f16(as<f16x8>(a), as<f16x8>(b), c, 0, 0, 0);
            else
                return __builtin_amdgcn_mfma_f32_32x32x16_bf16(as<bf16x8>(a), as<bf16x8>(b), c, 0, 0, 0);
        } else {
            if constexpr (P::half)
                return __builtin_amdgcn_mfma_f32_16x16x32_f16(as<f16x8>(a), as<f16x8>(b), c, 0, 0, 0);
            else
                return __builtin_amdgcn_mfma_f32_16x16x32_bf16(as<bf16x8>(a), as<bf16x8>(b), c, 0, 0, 0);
        }
    }
};

// Planes of a float32 value, each what is left of it times 2^8, rounded to nearest, so that what a product leaves out has no
// sign of its own; where that would round to infinity it is cut instead.  SMALL: values in [-1, 1], or no number.
template <bool SMALL = false>
__device__ __forceinline__ void split_planes(float f, bf16_t *p)
{
#pragma unroll
    for (int q = 0; q < 3; ++q) {
        bf16_t a = from_float<bf16_t>(f);
        if (!SMALL && (a.bits & 0x7fff) == 0x7f80 && fabsf(f) < INFINITY) a.bits = (uint16_t)(__float_as_uint(f) >> 16);
        p[q] = a;
        f = !SMALL && (a.bits & 0x7f80) == 0x7f80 ? 0.f : (f - to_float(a)) * 256.f;
    }
}

// Four values rounded to the 16-bit type of P, to nearest even.
template <typename P>
__device__ __forceinline__ s16x4 round4(f32x4 v)
{
    typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
    typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
    if constexpr (P::half) return __builtin_bit_cast(s16x4, __builtin_convertvector(v, f16x4));
    else return __builtin_bit_cast(s16x4, __builtin_convertvector(v, bf16x4));
}

// An operand: `rows` x `k` elements, 16 bits each.  Contiguous along k (element (r, k) at r * ld + k) or across it (at
// k * ld + r).  ld and the address allow 16-byte accesses; past `rows` or `k` everything up to the next multiple of 8 along the
// contiguous axis may be read and is zero, nothing beyond is touched.  Three planes lie in turns of 32 elements along the
// contiguous axis: element c of plane q at c / 32 * 96 + q * 32 + c % 32, and ld counts all three.
struct Operand {
    const void *at;
    int64_t ld;
};
// Elements of a row of n, all planes.
template <typename P> __host__ __device__ constexpr int64_t row_elements(int64_t n)
{
    return P::planes == 1 ? (n + 7) / 8 * 8 : (n + 31) / 32 * 96;
}

// Tiles of products that take float32 weights as they are.
constexpr int kRawWords = 128, kRawTokens = 64;

// What a launch computes with its tiles.
enum {
    kStats = 0,  // maxima and sums of the logits' exponentials
    kKeep = 1,   // the same, and the exponentials themselves, relative to their tile's maximum, in 32 bits: of float32 where P will be
                 // (32 of them in the first 128 of the 192 bytes that their planes will take), of 16-bit types beside it
    kProb = 2,   // P, from finished sums
    kOut = 3     // a gradient
};

struct Args {
    Operand a, b;
    int M, N, K;          // of the whole product
    int tiles_m, tiles_n;
    int splits, k_split;  // kOut: the reduction is cut into `splits` stretches of k_split (a multiple of the step)
    // logits: bias, targets, which stretch of the vocabulary this is
    const void *bias;
    int bias_type;
    const void *target;
    int target_wide;
    int64_t V, ignore;
    int v0;
    float *stats;         // kStats, kKeep: [tiles_m] [T][2] maximum and sum of exponentials, base 2
    float *picked;        // kStats, kKeep: [T] the target's logit
    // kProb (prob also kKeep)
    const float *lse;     // [T], base 2
    const float *row_scale;  // [T], or NULL: 1 for every counted row
    const float *row_power;  // float16, [T], or NULL: powers of two that rows have left to be multiplied with (kOut: of C)
    void *prob;           // [T] rows of ldp
    int64_t ldp;
    float *kept;          // kKeep of 16-bit types: [T] rows of ld_kept
    int64_t ld_kept;
    int prob_words;       // words of a row, a multiple of 32; zeros from M on
    float *bias_part;     // [tiles_n][ld of the piece]: sums over the rows of a tile, or NULL
    int ld_bias_part;
    void *bias_out;       // one tile holds all rows: the bias's gradient itself (times factor), or NULL
    uint32_t *arrived;    // kStats, kKeep: set to 0, for row_kernel
    // kOut
    float *slice;         // [splits][N][M] float, or NULL: final
    void *out;            // [N] rows of the operands' type, ldo apart
    int64_t ldo;
    const float *factor[2];  // what results are multiplied with, 1 value each, or NULL
    int n_store;          // rows of C that exist (N may be rounded up for the loads)
};

constexpr float kLog2e = 1.4426950408889634f;
// float16 holds probabilities times 2^15: the smallest that keeps all its bits is 2^-29 instead of 2^-14.  bfloat16 has the
// exponents of float32 and needs none.
constexpr float kProbScale = 32768.f;

// For terms of a sum whose largest is 1: one instruction, good to a unit in the last place; what is below 2^-126 becomes 0.
__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// All of 2^x's range; the few more instructions that takes only where a lane has an x below `least`, -126 or, in rows whose
// x are -inf throughout, -inf.
__device__ __forceinline__ void exp2_of_four(const float (&x)[4], float (&e)[4], float least = -126.f)
{
    if (__any(fminf(fminf(x[0], x[1]), fminf(x[2], x[3])) < least)) {
#pragma unroll
        for (int r = 0; r < 4; ++r) e[r] = exp2f(x[r]);
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) e[r] = exp2_of(x[r]);
    }
}

// A launch's tile: the workgroups of one XCD (they are dealt out in turn) get neighbouring tiles, in strips of kStrip along m,
// so that what they read at the same time fits its L2.
__device__ __forceinline__ void tile_of(int id, int tiles_m, int tiles_n, int splits, int *tm, int *tn, int *split)
{
    constexpr int kXcds = 8, kStrip = 8;
    const int tiles = tiles_m * tiles_n, even = tiles * splits / kXcds * kXcds;
    if (id < even) id = (id % kXcds) * (even / kXcds) + id / kXcds;
    *split = id / tiles;
    id -= *split * tiles;
    const int per_strip = kStrip * tiles_n;
    const int strip = id / per_strip, in = id - strip * per_strip;
    const int first = strip * kStrip, width = min(kStrip, tiles_m - first);
    *tn = in / width;
    *tm = first + in - *tn * width;
}

// 16 bytes per lane from a buffer to LDS: lane l's go to `lds` + 16 l.  An offset past 2^31 fetches zeros.  No register is
// written; whoever reads the LDS waits for the wave's own loads (vmcnt) and then for the workgroup's barrier.  The five wait
// states cover M0, which needs one, and a descriptor that a vector instruction might have written just before.
__device__ __forceinline__ void fetch(uint32_t offset, i32x4 buffer, uint32_t lds)
{
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
                 :: "v"(offset), "s"(buffer), "s"(lds) : "memory");
}
// The same, 4 bytes per lane, at `lds` + 4 l.
__device__ __forceinline__ void fetch_word(uint32_t offset, i32x4 buffer, uint32_t lds)
{
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tbuffer_load_dword %0, %1, 0 offen lds"
                 :: "v"(offset), "s"(buffer), "s"(lds) : "memory");
}
constexpr uint32_t kNothing = 0x80000000u;

__device__ __forceinline__ i32x4 buffer_at(uint64_t address)
{
    i32x4 r;
    r.x = __builtin_amdgcn_readfirstlane((int)(uint32_t)address);
    r.y = __builtin_amdgcn_readfirstlane((int)((uint32_t)(address >> 32) & 0xffffu));
    r.z = 0x7fffffff;
    r.w = 0x00020000;
    return r;
}

// A stage of one operand in LDS, ROWS x P::step, one plane after the other.
//   along k:  [row][k], rows of 128 (64) bytes, whose 16-byte pieces are exchanged by row, so that 16 lanes that read together
//             (0-3, 12-15, 20-23 and 24-27, and so on) meet all banks;
//   across:   [k][ROWS], its 32-byte pieces exchanged by k, so that the transposing reads that 32 lanes make together, of
//             k .. k + 3 and k + 8 .. k + 11 or of two neighbouring pieces of k .. k + 3, meet all banks.
template <typename P, int ROWS, bool ACROSS, int WAVES>
struct Tile {
    static constexpr int kStep = P::step, kPlanes = P::planes;
    static constexpr int bytes = ROWS * kStep * 2;           // of a plane
    static constexpr int fetches = bytes / 1024;             // 1 KB each
    static constexpr int mine = (fetches + WAVES - 1) / WAVES;  // of one wave
    static_assert((ROWS >= 64 || !ACROSS) && fetches % WAVES == 0, "every wave fetches the same number");
    static constexpr int kPieces = kStep / 8;                // of a row, along k

    uint32_t offset[mine];  // of this lane within the tile's first stage, or kNothing
    int k_at[mine];         // along: first k of this lane's piece; across: its k

    __device__ static __forceinline__ int swapped(int row) { return kPieces == 8 ? (row & 7) ^ (row >> 4 & 1) : row >> 1 & 3; }
    __device__ static __forceinline__ int swapped_across(int k)
    {
        if (Unit<P>::size == 32) return ROWS >= 128 ? (k & 3) << 1 : k & 2;
        return ROWS >= 128 ? (k & 3) | (k >> 1 & 4) : (k >> 1 & 1) | (k >> 2 & 2);
    }

    __device__ void init(const Operand &o, int rows_left, int wave)
    {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int i = 0; i < mine; ++i) {
            const int p = (wave * mine + i) * 64 + lane;  // 16-byte piece of the stage
            if constexpr (!ACROSS) {
                const int row = p / kPieces, piece = (p % kPieces) ^ swapped(row);
                k_at[i] = piece * 8;
                offset[i] = row < rows_left ? (uint32_t)(row * o.ld * 2 + piece * 16) : kNothing;
            } else {
                constexpr int per_k = ROWS / 8;
                const int k = p / per_k, piece = (p % per_k) ^ (swapped_across(k) << 1);
                k_at[i] = k;
                const int at = kPlanes == 1 ? piece * 16 : (piece >> 2) * 192 + (piece & 3) * 16;
                offset[i] = piece * 8 < rows_left ? (uint32_t)(k * o.ld * 2 + at) : kNothing;
            }
        }
    }
    // The wave's fetch `i` of a stage, of plane q; `k_left` of the reduction remain at this stage, whose element (0, 0) is at
    // `base`.
    __device__ __forceinline__ void one(uint64_t base, int k_left, uint32_t lds, int wave, int q, int i) const
    {
        fetch(k_at[i] < k_left ? offset[i] : kNothing, buffer_at(base + q * 64), lds + q * bytes + (wave * mine + i) * 1024);
    }
    __device__ __forceinline__ void stage(uint64_t base, int k_left, uint32_t lds, int wave) const
    {
#pragma unroll
        for (int q = 0; q < kPlanes; ++q)
#pragma unroll
            for (int i = 0; i < mine; ++i) one(base, k_left, lds, wave, q, i);
    }
    __device__ static __forceinline__ int64_t step_bytes(const Operand &o)
    {
        return ACROSS ? o.ld * kStep * 2 : kStep * kPlanes * 2;
    }
    // of rows before a tile: a multiple of 32 of them
    __device__ static __forceinline__ int64_t rows_bytes(const Operand &o, int rows)
    {
        return ACROSS ? (int64_t)rows * kPlanes * 2 : rows * o.ld * 2;
    }

    // Fragments of instruction `part` of the stage: unit rows from r0 (a multiple of unit), lane l gets row l % unit and eight k,
    // those from 8 (l / unit) on.
    __device__ static __forceinline__ s16x8 fragment(const char *lds, int r0, int part)
    {
        constexpr int U = Unit<P>::size, kDepth = Unit<P>::depth;
        const int lane = threadIdx.x & 63, g = lane / U;
        if constexpr (!ACROSS) {
            const int row = r0 + lane % U;
            return *(const s16x8 *)(lds + row * (kStep * 2) + (((part * (kDepth / 8) + g) ^ swapped(row)) << 4));
        } else {
            // 16 lanes read 4 k x 16 rows, 8 bytes each, and get them transposed
            typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
            const int i = lane & 15, k = part * kDepth + 8 * g + (i >> 2);
            const int piece = (r0 + lane % U) >> 4 ^ swapped_across(k);  // bit 2 of k, clear here, makes no difference
            const char *p = lds + k * ROWS * 2 + piece * 32 + (i & 3) * 8;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)p);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(p + 4 * ROWS * 2));
            s16x8 r;
            r.lo = lo;
            r.hi = hi;
            return r;
        }
    }
};

// A stage of float32 weights as they are, whose fragments are split into planes on their way out of LDS: for few tokens, where
// weights in planes would be written and read for little use.  Like a Tile, but for
//   along k:  [row][32], rows of 128 bytes, whose 16-byte pieces are exchanged by row;
//   across:   [k][ROWS], whose 64-byte pieces are exchanged by k / 8, so that the four groups of 16 lanes that read together
//             meet other banks.
// WIDTH floats a lane and fetch: four, where rows begin at multiples of 16 bytes and end at multiples of four floats, or one
// (28 tokens, 61003 words x 3405: the loss in 246 us, with planes written first 773).
template <int ROWS, bool ACROSS, int WAVES, int WIDTH>
struct RawTile {
    static constexpr int kStep = Split::step, kPlanes = 1;
    static constexpr int bytes = ROWS * kStep * 4, fetches = bytes / (256 * WIDTH), mine = fetches / WAVES;
    static_assert(fetches % WAVES == 0 && ROWS >= 64, "");

    // Fetches that are `kTurn` apart differ in what all lanes share: kShared rows (of 16 bytes along k, single floats across).
    // Fetch i of a wave has the floats from 64 WIDTH i on: of one float each, two rows, or half of a k.
    static constexpr int kTurn = WIDTH == 4 ? mine : ACROSS ? 2 : 4;
    uint32_t offset[kTurn];
    int k_at[kTurn];
    int rows_after;  // single floats along k: rows behind this lane's first one
    int64_t pitch;   // bytes

    __device__ static __forceinline__ int swapped(int row) { return row & 7; }
    __device__ static __forceinline__ int swapped_across(int k) { return (k >> 3 & 3) << 2; }

    __device__ void init(const Operand &o, int rows_left, int wave)
    {
        const int lane = threadIdx.x & 63;
        pitch = o.ld * 4;
        rows_after = rows_left - wave * mine * 2 - lane / 32;
#pragma unroll
        for (int i = 0; i < kTurn; ++i) {
            const int f = ((wave * mine + i) * 64 + lane) * WIDTH, p = f / 4, e = f % 4;  // float, 16-byte piece
            if constexpr (!ACROSS) {
                const int row = p / 8, piece = p % 8 ^ swapped(row);
                k_at[i] = piece * 4 + e;
                offset[i] = WIDTH == 1 || row < rows_left ? (uint32_t)(row * pitch + piece * 16 + e * 4) : kNothing;
            } else {
                const int k = p / (ROWS / 4), piece = p % (ROWS / 4) ^ swapped_across(k);
                k_at[i] = k;
                offset[i] = piece * 4 + e < rows_left ? (uint32_t)(k * pitch + piece * 16 + e * 4) : kNothing;
            }
        }
    }
    __device__ __forceinline__ void one(uint64_t base, int k_left, uint32_t lds, int wave, int, int i) const
    {
        const uint32_t to = lds + (wave * mine + i) * 256 * WIDTH;
        if constexpr (WIDTH == 4) {
            fetch(k_at[i] < k_left ? offset[i] : kNothing, buffer_at(base), to);
        } else if constexpr (ACROSS) {
            // a wave has mine / 2 whole k, whose pieces are exchanged alike
            static_assert(ROWS == 128 && mine / 2 == 8, "");
            const int k = wave * (mine / 2) + i / 2;
            fetch_word(k < k_left ? offset[i % 2] : kNothing, buffer_at(base + i / 2 * pitch), to);
        } else {
            // rows 2 i on: the exchange comes again after eight of them
            const bool real = 2 * i < rows_after && k_at[i % 4] < k_left;
            fetch_word(real ? offset[i % 4] : kNothing, buffer_at(base + i / 4 * 8 * pitch), to);
        }
    }
    __device__ __forceinline__ void stage(uint64_t base, int k_left, uint32_t lds, int wave) const
    {
#pragma unroll
        for (int i = 0; i < mine; ++i) one(base, k_left, lds, wave, 0, i);
    }
    __device__ static __forceinline__ int64_t step_bytes(const Operand &o) { return ACROSS ? o.ld * kStep * 4 : kStep * 4; }
    __device__ static __forceinline__ int64_t rows_bytes(const Operand &o, int rows)
    {
        return ACROSS ? (int64_t)rows * 4 : rows * o.ld * 4;
    }

    // 16 rows from r0 on, lane l's being row l % 16 and the eight k from 8 (l / 16) on
    __device__ static __forceinline__ void load(const char *lds, int r0, float (&x)[8])
    {
        const int lane = threadIdx.x & 63, g = lane / 16, row = r0 + lane % 16;
        if constexpr (!ACROSS) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const f32x4 v = *(const f32x4 *)(lds + row * 128 + (((2 * g + half) ^ swapped(row)) << 4));
#pragma unroll
                for (int e = 0; e < 4; ++e) x[half * 4 + e] = v[e];
            }
        } else {
            const char *p = lds + g * 8 * ROWS * 4 + ((row / 4 ^ swapped_across(g * 8)) * 16 + row % 4 * 4);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = *(const float *)(p + e * ROWS * 4);
        }
    }
    // Planes of two of them.  EXACT: of all values; else of those below kLimit, and `top` becomes the largest.
    static constexpr float kLimit = 0x1.fep127f;  // what rounds to infinity, and infinities
    template <bool EXACT>
    __device__ static __forceinline__ void split(const float (&x)[8], int e, s16x8 (&planes)[3], float &top)
    {
        float a = x[e], b = x[e + 1];
        if constexpr (EXACT) {
            bf16_t p[3], q[3];
            split_planes(a, p), split_planes(b, q);
#pragma unroll
            for (int k = 0; k < 3; ++k) planes[k][e] = (short)p[k].bits, planes[k][e + 1] = (short)q[k].bits;
            return;
        }
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        top = fmaxf(top, fmaxf(fabsf(a), fabsf(b)));
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            const uint32_t two = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
            planes[k][e] = (short)two, planes[k][e + 1] = (short)(two >> 16);
            a = (a - __uint_as_float(two << 16)) * 256.f, b = (b - __uint_as_float(two & 0xffff0000u)) * 256.f;
        }
    }
};

__device__ __forceinline__ float bias_at(const Args &a, int v)
{
    if (!a.bias) return 0.f;
    if (a.bias_type == DS_F32) return ((const float *)a.bias)[v];
    if (a.bias_type == DS_BF16) return to_float(((const bf16_t *)a.bias)[v]);
    return to_float(((const f16_t *)a.bias)[v]);
}

__device__ __forceinline__ int64_t target_at(const Args &a, int t)
{
    return a.target_wide ? ((const int64_t *)a.target)[t] : (int64_t)((const int32_t *)a.target)[t];
}

// What sums of probabilities are multiplied with on their way out, and what probabilities are: the loss's gradient times a row's
// share belongs to the former if it is a number, else to the rows that count, so that it makes nothing of the others' zeros.
__device__ __forceinline__ float both_factors(const float *const *f) { return (f[0] ? *f[0] : 1.f) * (f[1] ? *f[1] : 1.f); }
__device__ __forceinline__ float factor_of(const float *const *f)
{
    const float all = both_factors(f);
    return fabsf(all) < INFINITY ? all : 1.f;
}
__device__ __forceinline__ float prob_factor_of(const float *const *f)
{
    const float all = both_factors(f);
    return fabsf(all) < INFINITY ? 1.f : all;
}
template <typename P>
__device__ __forceinline__ float out_factor(const float *const *f)
{
    return factor_of(f) * (P::half ? 1.f / kProbScale : 1.f);
}
template <typename P> struct ElementOf { typedef bf16_t type; };
template <> struct ElementOf<F16> { typedef f16_t type; };
template <> struct ElementOf<Split> { typedef float type; };

// Until all but `in_flight` of this wave's fetches have arrived and all its reads of LDS, and then until every wave's have.
template <int in_flight>
__device__ __forceinline__ void wait_for_stage()
{
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "i"(in_flight) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// LDS of a workgroup: the stages, and what the epilogue of the logits needs to know of its words and tokens, fetched before
// the products start (one load after another behind them took half of a short reduction's time).
template <typename P, int BM, int BN, int STAGES, bool RAW = false>
constexpr int kStagesBytes = STAGES * P::step * (RAW ? BM * 4 + P::planes * BN * 2 : P::planes * (BM + BN) * 2);
template <int BM, int BN>
struct Known {
    float bias[BM];   // times log2 e; -inf for words past the end, which leave nothing that way
    int want[BN];     // the target, counted from the tile's first word, where it lies in the tile; else far below 0
    float lse[BN];    // +inf for rows that do not count: theirs are probabilities of 0
    float scale[BN];
    float power[BN];
};
// Rows that leave together, what one of them takes, and whether the waves' maxima and sums find a place behind them in the
// stages (256 x 256 tiles' exponentials fill those).
template <typename P, int WN> constexpr int kRowsLeaving = WN * Unit<P>::size;
template <typename P, int BM, int KIND> constexpr int kRowBytes = KIND == kOut || (KIND == kKeep && P::planes == 1) ? BM * 4 : BM * P::planes * 2;
template <typename P, int BM, int BN, int WM, int WN, int KIND, int STAGES, bool RAW>
constexpr bool kRoomBehind = KIND == kStats || kRowsLeaving<P, WN> * kRowBytes<P, BM, KIND> + WM * BN * 8 <= kStagesBytes<P, BM, BN, STAGES, RAW>;
template <typename P, int BM, int BN, int WM, int WN, int KIND, int STAGES, bool RAW = false>
constexpr int kLdsBytes = kStagesBytes<P, BM, BN, STAGES, RAW> + (KIND != kOut ? (int)sizeof(Known<BM, BN>) : 0) +
                          (KIND == kKeep && !kRoomBehind<P, BM, BN, WM, WN, KIND, STAGES, RAW> ? WM * BN * 8 : 0) +
                          (P::planes > 1 ? 16 : 0);

// Results on their way out: rows of COLS elements gathered in LDS, whose 16-byte pieces are exchanged by row, so that lanes
// that each hold a few neighbours of another row do not meet in a bank; from there every row leaves as one stretch.  (Stored
// from the registers, eight bytes here and there, a tile of 256 x 256 took some 25 us.)  Rows may begin anywhere: 50021 x 2049
// bfloat16 gradients of four tokens leave in 73 us (120 by elements), 2048 of them in 60.
template <typename S, int COLS>
struct Gather {
    static constexpr int kPer = 16 / sizeof(S), kPieces = COLS / kPer;
    static constexpr int kMask = (kPieces & -kPieces) < 32 ? (kPieces & -kPieces) - 1 : 31;

    __device__ static __forceinline__ char *at(char *lds, int row, int col)
    {
        const int piece = col / kPer ^ (row & kMask);
        return lds + (row * kPieces + piece) * 16 + col % kPer * (int)sizeof(S);
    }
    // `row_at(r)` is where row r goes, or NULL; `cols` of it exist, and of every TURN only the first FILLED
    template <int THREADS, int FILLED = 1, int TURN = 1, typename ROW>
    __device__ static __forceinline__ void leave(char *lds, int rows, int cols, ROW row_at)
    {
        for (int i = threadIdx.x; i < rows * kPieces; i += THREADS) {
            const int row = i / kPieces, col = i % kPieces * kPer;
            S *to = row_at(row);
            if (!to || col >= cols || col % TURN >= FILLED) continue;
            to += col;
            const Vec<S, kPer> v = *(const Vec<S, kPer> *)at(lds, row, col);
            if (col + kPer <= cols && (uintptr_t)to % 16 == 0) {
                *(Vec<S, kPer> *)to = v;
            } else if (col + kPer <= cols) {
                // wherever it lies; the compiler is kept from seeing the same values stored on all three paths, for which it
                // finds common pieces
                typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
                u32x4 w = __builtin_bit_cast(u32x4, v);
                asm("" : "+v"(w));
                __builtin_memcpy(to, &w, 16);
            } else {
#pragma unroll
                for (int e = 0; e < kPer; ++e)
                    if (col + e < cols) to[e] = v.v[e];
            }
        }
    }
};

// Sums of N values over the lanes that differ in the bits below 2 O; returns which of them this lane has, from v[0] on.
template <int O, int N, int ALL>
__device__ __forceinline__ int spread_sums(float (&v)[ALL], int lane)
{
    if constexpr (O == 0) {
        return 0;
    } else if constexpr (N > 1) {
        const bool upper = lane & O;
#pragma unroll
        for (int k = 0; k < N / 2; ++k) {
            const float away = upper ? v[k] : v[k + N / 2], kept = upper ? v[k + N / 2] : v[k];
            v[k] = kept + __shfl_xor(away, O);
        }
        return (upper ? N / 2 : 0) + spread_sums<O / 2, N / 2>(v, lane);
    } else {
        v[0] += __shfl_xor(v[0], O);
        return spread_sums<O / 2, 1>(v, lane);
    }
}

// One tile of a product, by a whole workgroup; `block` counts the product's workgroups.
//
// Operands go from memory to LDS without registers, two stages and more ahead; a wave holds up to 128 x 64 results.  Fragments
// are read and stages fetched between rows of products, a few each: with all of them behind the barrier the matrix cores were
// busy 55 % of the cycles instead of 70 to 85 (4.0 instead of 3.2 ms for the scores above).  32 x 32 instructions take half as
// many issues as 16 x 16 ones at the same rate; float32 keeps the smaller ones, whose partial sums of the planes fit.
template <typename P, int BM, int BN, int WM, int WN, bool A_ACROSS, bool B_ACROSS, int KIND, int STAGES, int RAW = 0>
__device__ __forceinline__ void product_tile(const Args &g, const int block, char *lds)
{
    using U = Unit<P>;
    constexpr int WAVES = WM * WN, MT = BM / WM / U::size, NT = BN / WN / U::size, NP = P::planes;
    constexpr int kStep = P::step;
    static_assert(!RAW || NP == 3, "");
    using TA = typename std::conditional<(RAW > 0), RawTile<BM, A_ACROSS, WAVES, RAW ? RAW : 4>, Tile<P, BM, A_ACROSS, WAVES>>::type;
    using TB = Tile<P, BN, B_ACROSS, WAVES>;
    constexpr int kBytesA = TA::kPlanes * TA::bytes, kStageBytes = kBytesA + NP * TB::bytes;
    constexpr int kFetchesA = TA::kPlanes * TA::mine, kInFlight = kFetchesA + NP * TB::mine;  // loads of one stage and wave
    static_assert(STAGES * kStageBytes == kStagesBytes<P, BM, BN, STAGES, (RAW > 0)>, "");
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int wm = wave % WM, wn = wave / WM;

    int tm, tn, split;
    tile_of(block, g.tiles_m, g.tiles_n, g.splits, &tm, &tn, &split);
    const int m0 = tm * BM, n0 = tn * BN;
    const int k_from = split * g.k_split, k_to = min(g.K, k_from + g.k_split);
    const int steps = (k_to - k_from + kStep - 1) / kStep;

    TA ta;
    TB tb;
    ta.init(g.a, g.M - m0, wave);
    tb.init(g.b, g.N - n0, wave);
    const int64_t a_step = TA::step_bytes(g.a), b_step = TB::step_bytes(g.b);
    uint64_t a_at = (uint64_t)g.a.at + TA::rows_bytes(g.a, m0) + k_from / kStep * a_step;
    uint64_t b_at = (uint64_t)g.b.at + TB::rows_bytes(g.b, n0) + k_from / kStep * b_step;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;

    int k_left = k_to - k_from;  // of the next stage to fetch
    auto fetch_stage = [&](int slot) {
        const uint32_t to = lds0 + slot * kStageBytes;
        ta.stage(a_at, k_left, to, wave);
        tb.stage(b_at, k_left, to + kBytesA, wave);
        a_at += a_step, b_at += b_step, k_left -= kStep;
    };

    typename U::Result acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int r = 0; r < 4 * U::groups; ++r) acc[i][j][r] = 0.f;

    Known<BM, BN> &known = *(Known<BM, BN> *)(lds + kStagesBytes<P, BM, BN, STAGES, (RAW > 0)>);
    static_assert(BM <= WAVES * 64 && BN <= WAVES * 64, "a thread per word and token");
    constexpr int kNowhere = -(1 << 20);
    float bias = -INFINITY, lse = INFINITY, scale = 0.f, power = 1.f;
    int want = kNowhere;
    if constexpr (KIND != kOut) {
        const int m = m0 + threadIdx.x, n = n0 + threadIdx.x;
        if (threadIdx.x < BM && m < g.M) bias = bias_at(g, g.v0 + m) * kLog2e;
        if (threadIdx.x < BN && n < g.N) {
            const int64_t y = target_at(g, n), here = y - g.v0 - m0;
            if (here >= 0 && here < BM && m0 + here < g.M) want = (int)here;
            if constexpr (KIND == kProb) {
                if (y != g.ignore) {
                    lse = g.lse[n];
                    scale = y < 0 || y >= g.V ? NAN : g.row_scale ? g.row_scale[n] : prob_factor_of(g.factor);
                    if (P::half && g.row_power) power = g.row_power[n];
                } else {
                    want = kNowhere;
                }
            }
        }
    }

    int *const met_nan = (int *)(lds + kLdsBytes<P, BM, BN, WM, WN, KIND, STAGES, (RAW > 0)>) - 1;  // of float32: a result is NaN
    auto keep_known = [&] {
        if (NP > 1 && threadIdx.x == 0) *met_nan = 0;
        if constexpr (KIND != kOut) {
            if (threadIdx.x < BM) known.bias[threadIdx.x] = bias;
            if (threadIdx.x < BN)
                known.want[threadIdx.x] = want, known.lse[threadIdx.x] = lse, known.scale[threadIdx.x] = scale;
            if (P::half && KIND == kProb && threadIdx.x < BN) known.power[threadIdx.x] = power;
        }
    };

    // Stages past the end are fetched too, as zeros (k_left <= 0 fetches nothing): the number of loads in flight is the same
    // in every step, and nothing past the operands is read.
    int slot = 0;
    if constexpr (NP == 1) {
        // While the products of one half of a stage run, the fragments of the next half are read: the second half's between
        // the first's products, the next stage's first half between the second's.  In the middle, where every wave has read
        // the whole stage, its slot is fetched anew, one fetch after each row of products.
        constexpr int kParts = kStep / U::depth / 2, kRows = kParts * MT, kFragments = kParts * (MT + NT);
        constexpr int kPerRow = (kFragments * 4 + kRows * 3 - 1) / (kRows * 3);  // read in the first three quarters of the rows
        constexpr int kFetches = TA::mine + TB::mine, kFetchesPerRow = (kFetches + kRows - 1) / kRows;
        s16x8 a0[kParts][MT], b0[kParts][NT], a1[kParts][MT], b1[kParts][NT];
        auto read = [&](int from, int half, int n, s16x8 (&fa)[kParts][MT], s16x8 (&fb)[kParts][NT]) {
            const char *at = lds + from * kStageBytes;
            const int p = n / (MT + NT), k = n % (MT + NT);
            if (n >= kFragments) return;
            if (k < NT) fb[p][k] = TB::fragment(at + TA::bytes, (wn * NT + k) * U::size, half * kParts + p);
            else fa[p][k - NT] = TA::fragment(at, (wm * MT + k - NT) * U::size, half * kParts + p);
        };
        auto multiply = [&](int row, const s16x8 (&fa)[kParts][MT], const s16x8 (&fb)[kParts][NT]) {
            const int p = row / MT, i = row % MT;
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = U::multiply(fa[p][i], fb[p][j], acc[i][j]);
        };
#pragma unroll
        for (int s = 0; s < STAGES; ++s) fetch_stage(s);
        keep_known();
        wait_for_stage<(STAGES - 1) * kInFlight>();
#pragma unroll
        for (int n = 0; n < kFragments; ++n) read(0, 0, n, a0, b0);
        for (int s = 0; s < steps; ++s) {
#pragma unroll
            for (int row = 0; row < kRows; ++row) {
                multiply(row, a0, b0);
#pragma unroll
                for (int n = 0; n < kPerRow; ++n) read(slot, 1, row * kPerRow + n, a1, b1);
                __builtin_amdgcn_sched_barrier(0);
            }
            wait_for_stage<(STAGES - 2) * kInFlight>();
            const uint32_t to = lds0 + slot * kStageBytes;
            slot = slot + 1 == STAGES ? 0 : slot + 1;
#pragma unroll
            for (int row = 0; row < kRows; ++row) {
                multiply(row, a1, b1);
#pragma unroll
                for (int f = row * kFetchesPerRow; f < (row + 1) * kFetchesPerRow && f < kFetches; ++f) {
                    if (f < TA::mine) ta.one(a_at, k_left, to, wave, 0, f);
                    else tb.one(b_at, k_left, to + TA::bytes, wave, 0, f - TA::mine);
                }
#pragma unroll
                for (int n = 0; n < kPerRow; ++n) read(slot, 0, row * kPerRow + n, a0, b0);
                __builtin_amdgcn_sched_barrier(0);
            }
            a_at += a_step, b_at += b_step, k_left -= kStep;
        }
    } else {
        float top = 0.f;  // of weights that are split here
        // from the beginning again, for weights that the quick split does not do
        auto restart = [&] {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __syncthreads();
            const int64_t done = (int64_t)(steps + STAGES);
            a_at -= done * a_step, b_at -= done * b_step, k_left = k_to - k_from, slot = 0;
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        };
        auto products = [&](auto exact) {
            // Rows of tiles that are multiplied together: the six products of a tile follow each other, so four tiles at least have
            // to take turns.  While one such group is multiplied the next one's fragments of A are read; during the last group of a
            // stage, whose fragments are all there by then, the next stage's first ones, and its own slot is fetched anew.
            constexpr int G = NT >= 4 || MT == 1 ? 1 : 2, kGroups = MT / G;
            static_assert(MT % G == 0 && (kGroups == 1 || kGroups % 2 == 0), "");
            constexpr int kTurns = 6, kFetches = kInFlight, kReads = NP * (NT + G);
            s16x8 b0[NP][NT], b1[NP][NT], a0[G][NP], a1[G][NP], turn[G][NP];
            float whole[G][8];  // of weights that are split here
            auto read_a = [&](int from, int group, int n, s16x8 (&fa)[G][NP]) {
                const int i = n / NP, p = n % NP;
                const char *at = lds + from * kStageBytes;
                if constexpr (RAW) {
                    if (p == 0) TA::load(at, (wm * MT + group * G + i) * U::size, whole[i]);
                } else {
                    fa[i][p] = TA::fragment(at + p * TA::bytes, (wm * MT + group * G + i) * U::size, 0);
                }
            };
            // two of the eight in turn t, 1 to 4
            auto split_a = [&](int t, s16x8 (&fa)[G][NP]) {
                if constexpr (RAW)
                    if (t >= 1 && t <= 4)
#pragma unroll
                        for (int i = 0; i < G; ++i) TA::template split<decltype(exact)::value>(whole[i], (t - 1) * 2, fa[i], top);
            };
            auto read_b = [&](int from, int n, s16x8 (&fb)[NP][NT]) {
                const int p = n / NT, j = n % NT;
                fb[p][j] = TB::fragment(lds + from * kStageBytes + kBytesA + p * TB::bytes, (wn * NT + j) * U::size, 0);
            };
            // The products of 2^-16, the largest ones while those are made 2^-8, then the products of 2^-8; between(0) ..
            // between(kTurns - 1) in between.  What they amount to joins the result during the first turns of the next group (of
            // this one, where it is the only one): the matrix cores do not wait for either.
            f32x4 low[2][G][NT];
            auto join = [&](int group, int i, int j) {
                f32x4 &c = acc[group * G + i][j];
#pragma unroll
                for (int r = 0; r < 4; ++r) c[r] = fmaf(low[group % 2][i][j][r], 1.f / 256, c[r]);
            };
            auto multiply = [&](int group, const s16x8 (&fa)[G][NP], const s16x8 (&fb)[NP][NT], auto between) {
                f32x4(&mine)[G][NT] = low[group % 2];
                const int last = (group + kGroups - 1) % kGroups;
                auto add = [&](int p, int q, auto besides) {
#pragma unroll
                    for (int i = 0; i < G; ++i)
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            mine[i][j] = U::multiply(fa[i][p], fb[q][j], mine[i][j]);
                            besides(i, j);
                        }
                };
                auto nothing = [](int, int) {};
#pragma unroll
                for (int i = 0; i < G; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j) mine[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
                add(1, 1, [&](int i, int j) {
                    if (kGroups > 1) join(last, i, j);
                });
                between(0);
                add(0, 2, nothing), between(1);
                add(2, 0, nothing), between(2);
#pragma unroll
                for (int i = 0; i < G; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        f32x4 &c = acc[group * G + i][j];
                        c = U::multiply(fa[i][0], fb[0][j], c);
                        mine[i][j] *= 1.f / 256;
                    }
                between(3);
                add(0, 1, nothing), between(4);
                add(1, 0, nothing), between(5);
                if (kGroups == 1)
#pragma unroll
                    for (int i = 0; i < G; ++i)
#pragma unroll
                        for (int j = 0; j < NT; ++j) join(group, i, j);
            };
            auto step = [&](s16x8 (&fb)[NP][NT], s16x8 (&fa)[G][NP], s16x8 (&next_b)[NP][NT], s16x8 (&next_a)[G][NP]) {
#pragma unroll
                for (int k = 0; k + 1 < kGroups; ++k)
                    multiply(k, k % 2 ? turn : fa, fb, [&](int t) {
                        if (t == 0)
#pragma unroll
                            for (int n = 0; n < G * NP; ++n) read_a(slot, k + 1, n, k % 2 ? fa : turn);
                        split_a(t, k % 2 ? fa : turn);
                        __builtin_amdgcn_sched_barrier(0);
                    });
                wait_for_stage<(STAGES - 2) * kInFlight>();
                const uint32_t to = lds0 + slot * kStageBytes;
                slot = slot + 1 == STAGES ? 0 : slot + 1;
                multiply(kGroups - 1, kGroups > 1 ? turn : fa, fb, [&](int t) {
                    // a share of the fetches and of the reads, the latter in the first five turns
#pragma unroll
                    for (int f = 0; f < kFetches; ++f) {
                        if (f * kTurns / kFetches != t) continue;
                        if (f < kFetchesA) ta.one(a_at, k_left, to, wave, f / TA::mine, f % TA::mine);
                        else tb.one(b_at, k_left, to + kBytesA, wave, (f - kFetchesA) / TB::mine, (f - kFetchesA) % TB::mine);
                    }
#pragma unroll
                    for (int n = 0; n < kReads; ++n) {
                        if (n * (kTurns - 1) / kReads != t) continue;
                        if (n < G * NP) read_a(slot, 0, n, next_a);
                        else read_b(slot, n - G * NP, next_b);
                    }
                    split_a(t, next_a);
                    __builtin_amdgcn_sched_barrier(0);
                });
                a_at += a_step, b_at += b_step, k_left -= kStep;
            };
            if constexpr (decltype(exact)::value) restart();
#pragma unroll
            for (int s = 0; s < STAGES; ++s) fetch_stage(s);
            keep_known();
            wait_for_stage<(STAGES - 1) * kInFlight>();
#pragma unroll
            for (int n = 0; n < G * NP; ++n) read_a(0, 0, n, a0);
#pragma unroll
            for (int t = 1; t <= 4; ++t) split_a(t, a0);
#pragma unroll
            for (int n = 0; n < NP * NT; ++n) read_b(0, n, b0);
            if (kGroups > 1)
#pragma unroll
                for (int i = 0; i < G; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j) low[(kGroups - 1) % 2][i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
            for (int s = 0; s < steps; s += 2) {
                step(b0, a0, b1, a1);
                if (s + 1 < steps) step(b1, a1, b0, a0);
            }
            if (kGroups > 1)
#pragma unroll
                for (int i = 0; i < G; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j) join(kGroups - 1, i, j);
        };
        products(std::false_type());
        if constexpr (RAW)
            if (__syncthreads_or(top >= TA::kLimit)) products(std::true_type());
    }
    if constexpr (NP > 1) {
        bool odd = false;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
                odd |= __builtin_isunordered(acc[i][j][0], acc[i][j][1]) || __builtin_isunordered(acc[i][j][2], acc[i][j][3]);
        if (odd) *met_nan = 1;
    }
    // nothing of this wave is on its way to LDS any more, and nobody reads it
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __syncthreads();
    if constexpr (NP > 1) {
        // An infinity times a lower plane of 0, or of the other sign than its value, makes a result NaN that may be infinite.
        // The largest planes have the values' signs, zeros and infinities: their product alone says which it is.  A row of
        // the wave's tiles at a time, for the whole workgroup where a lane has met one, so that all of it fetches.  Looking for
        // them takes 0.2 us of a launch of 12 (with this code in the way of what follows 0.4); a step of 2048 x 1024 over 32768
        // words takes 4.3 ms instead of 2.6 with a NaN in one token, 5.3 with one in every word.
        if (__builtin_expect(*met_nan, 0)) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                f32x4 largest[NT];
#pragma unroll
                for (int j = 0; j < NT; ++j) largest[j] = f32x4{0.f, 0.f, 0.f, 0.f};
                a_at = (uint64_t)g.a.at + TA::rows_bytes(g.a, m0) + k_from / kStep * a_step;
                b_at = (uint64_t)g.b.at + TB::rows_bytes(g.b, n0) + k_from / kStep * b_step;
                k_left = k_to - k_from;
#pragma unroll 1
                for (int s = 0; s < steps; ++s) {
#pragma unroll
                    for (int f = 0; f < TA::mine; ++f) ta.one(a_at, k_left, lds0, wave, 0, f);
#pragma unroll
                    for (int f = 0; f < TB::mine; ++f) tb.one(b_at, k_left, lds0 + kBytesA, wave, 0, f);
                    a_at += a_step, b_at += b_step, k_left -= kStep;
                    wait_for_stage<0>();
                    s16x8 fa;
                    if constexpr (RAW) {
                        float x[8];
                        TA::load(lds, (wm * MT + i) * U::size, x);
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            bf16_t planes[3];
                            split_planes(x[e], planes);
                            fa[e] = (short)planes[0].bits;
                        }
                    } else {
                        fa = TA::fragment(lds, (wm * MT + i) * U::size, 0);
                    }
#pragma unroll
                    for (int j = 0; j < NT; ++j)
                        largest[j] = U::multiply(fa, TB::fragment(lds + kBytesA, (wn * NT + j) * U::size, 0), largest[j]);
                    wait_for_stage<0>();
                }
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (acc[i][j][r] != acc[i][j][r]) acc[i][j][r] = largest[j][r];
            }
        }
    }

    // This lane's results: I counts its groups of four neighbouring m, j its n.
    constexpr int MG = MT * U::groups;
    const int m_in = wm * MT * U::size + U::lane_m(lane), n_in = wn * NT * U::size + lane % U::size;  // in the tile
    auto m_of = [](int I) constexpr { return I / U::groups * U::size + U::group_m(I % U::groups); };
    auto value = [&](int I, int j, int r) -> float { return acc[I / U::groups][j][I % U::groups * 4 + r]; };
    float *fl = (float *)lds;
    // a logit, base 2
    auto logit = [&](int I, int j, int r) -> float { return fmaf(value(I, j, r), kLog2e, known.bias[m_in + m_of(I) + r]); };
    constexpr int kRowsOut = kRowsLeaving<P, WN>, kThreads = WAVES * 64;  // one j of every wave
    static_assert(KIND == kStats || kRowsOut * kRowBytes<P, BM, KIND> <= kStagesBytes<P, BM, BN, STAGES, (RAW > 0)>, "");
    auto n_of = [](int row, int j) { return (row / U::size * NT + j) * U::size + row % U::size; };
    const int row_out = wn * U::size + lane % U::size;
    // Four neighbouring probabilities to their place among the rows that leave.  Here they are rounded to the operands' type (of
    // float32 nothing is lost in three planes): the second product's other operand has no more bits either, and each rounding is
    // independent of the others.  Against 64 bits the gradients of 2048 tokens over 32768 words are 0.0017 of their norm off in
    // bfloat16, as a float32 computation rounded once at its end is; over 64 words, where more than the targets' probabilities
    // count, 0.0020 (float16 0.00026 and 0.00021).  Two planes of P would halve the rate of both gradients' products.
    auto put_prob = [&](int I, float (&p)[4]) {
        typedef Gather<uint16_t, BM * NP> Out;
        const int m = m_in + m_of(I);
        if constexpr (NP == 1 && KIND == kKeep) {
            *(f32x4 *)Gather<float, BM>::at(lds, row_out, m) = f32x4{p[0], p[1], p[2], p[3]};
        } else if constexpr (KIND == kKeep) {
            *(f32x4 *)Out::at(lds, row_out, (m >> 5) * 96 + (m & 31) * 2) = f32x4{p[0], p[1], p[2], p[3]};
        } else if constexpr (NP == 1) {
            *(s16x4 *)Out::at(lds, row_out, m) = round4<P>(f32x4{p[0], p[1], p[2], p[3]} * (P::half ? kProbScale : 1.f));
        } else {
            bf16_t planes[4][3];
#pragma unroll
            for (int r = 0; r < 4; ++r) split_planes<true>(p[r], planes[r]);
#pragma unroll
            for (int q = 0; q < NP; ++q) {
                const Vec<bf16_t, 4> o{{planes[0][q], planes[1][q], planes[2][q], planes[3][q]}};
                *(Vec<bf16_t, 4> *)Out::at(lds, row_out, (m >> 5) * 96 + q * 32 + (m & 31)) = o;
            }
        }
    };
    auto leave_prob = [&](int j) {
        __syncthreads();
        if constexpr (NP == 1 && KIND == kKeep) {
            Gather<float, BM>::template leave<kThreads>(lds, kRowsOut, g.prob_words - m0, [&](int row) -> float * {
                const int t = n0 + n_of(row, j);
                return t < g.N ? g.kept + t * g.ld_kept + m0 : nullptr;
            });
        } else {
            constexpr int kFilled = KIND == kKeep ? 64 : 96;  // of three planes' place
            Gather<uint16_t, BM * NP>::template leave<kThreads, kFilled, 96>(lds, kRowsOut, (g.prob_words - m0) * NP, [&](int row) -> uint16_t * {
                const int t = n0 + n_of(row, j);
                return t < g.N ? (uint16_t *)g.prob + t * g.ldp + m0 * NP : nullptr;
            });
        }
        __syncthreads();
    };
    if constexpr (KIND == kStats || KIND == kKeep) {
        if (block == 0 && threadIdx.x == 0) *g.arrived = 0;
        float tops[NT];
        auto tops_of = [&](int j) {
            const int at = known.want[n_in + j * U::size] - m_in;  // where the target lies behind this lane's first word
            float top = -INFINITY;
#pragma unroll
            for (int I = 0; I < MG; ++I) {
                float s[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[r] = logit(I, j, r);
                    top = fmaxf(top, s[r]);  // what is no number shows in the sum
                }
                if ((unsigned)(at - m_of(I)) < 4u)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (at == m_of(I) + r) g.picked[n0 + n_in + j * U::size] = s[r];
            }
            return top;
        };
        // exponentials relative to `top`, and their sum over this lane's words; a column of nothing but -inf keeps a sum of 0
        auto sum_of = [&](int j, float top) {
            const float base = top == -INFINITY ? 0.f : top;
            float sum = 0.f;
#pragma unroll
            for (int I = 0; I < MG; ++I) {
                float x[4], e[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) x[r] = logit(I, j, r) - base;
                // a sum does not notice what the instruction by itself leaves out, what is kept has it
                if constexpr (KIND == kKeep) exp2_of_four(x, e);
                else
#pragma unroll
                    for (int r = 0; r < 4; ++r) e[r] = exp2_of(x[r]);
#pragma unroll
                for (int r = 0; r < 4; ++r) sum += e[r];
                if constexpr (KIND == kKeep) put_prob(I, e);
            }
            return sum;
        };
        // a place behind the rows on their way out, where other waves' results wait
        constexpr bool kRoom = kRoomBehind<P, BM, BN, WM, WN, KIND, STAGES, (RAW > 0)>;
        float2 *const others = kRoom ? (float2 *)(lds + kStagesBytes<P, BM, BN, STAGES, (RAW > 0)>) - WM * BN : (float2 *)(&known + 1);
        if constexpr (KIND == kKeep) {
            // the tile's maximum first: what is kept is relative to it
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                tops[j] = tops_of(j);
#pragma unroll
                for (int o = U::size; o < 64; o <<= 1) tops[j] = fmaxf(tops[j], __shfl_xor(tops[j], o));
                if (lane < U::size) others[wm * BN + (wn * NT + j) * U::size + lane].x = tops[j];
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int w = 0; w < WM; ++w) tops[j] = fmaxf(tops[j], others[w * BN + n_in + j * U::size].x);
            __syncthreads();
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            float top = KIND == kKeep ? tops[j] : tops_of(j);
            float sum = sum_of(j, top);
#pragma unroll
            for (int o = U::size; o < 64; o <<= 1) {
                const float top2 = __shfl_xor(top, o), sum2 = __shfl_xor(sum, o);
                const float both = fmaxf(top, top2);
                sum = both == -INFINITY ? sum + sum2 : sum * exp2_of(top - both) + sum2 * exp2_of(top2 - both);
                top = both;
            }
            if (lane < U::size) others[wm * BN + (wn * NT + j) * U::size + lane] = float2{top, sum};
            if constexpr (KIND == kKeep) leave_prob(j);
        }
        __syncthreads();
        for (int c = threadIdx.x; c < BN; c += WAVES * 64) {
            if (n0 + c >= g.N) continue;
            float top = others[c].x, sum = others[c].y;
#pragma unroll
            for (int w = 1; w < WM; ++w) {
                const float top2 = others[w * BN + c].x, sum2 = others[w * BN + c].y;
                const float both = fmaxf(top, top2);
                sum = both == -INFINITY ? sum + sum2 : sum * exp2_of(top - both) + sum2 * exp2_of(top2 - both);
                top = both;
            }
            ((float2 *)g.stats)[(int64_t)tm * g.N + n0 + c] = float2{top, sum};
        }
    }
    if constexpr (KIND == kProb) {
        float over_n[MG * 4];  // sums over this lane's rows, for the bias
#pragma unroll
        for (int k = 0; k < MG * 4; ++k) over_n[k] = 0.f;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const float lse = known.lse[n_in + j * U::size], scale = known.scale[n_in + j * U::size];
            const float power = P::half ? known.power[n_in + j * U::size] : 1.f;
            const float least = lse == INFINITY ? -INFINITY : -126.f;
            const bool counts = !(lse == INFINITY && scale == 0.f);  // else nothing is left, also of infinite weights times 0
            const int at = known.want[n_in + j * U::size] - m_in;
#pragma unroll
            for (int I = 0; I < MG; ++I) {
                float x[4], p[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) x[r] = logit(I, j, r) - lse;
                exp2_of_four(x, p, least);
                if ((unsigned)(at - m_of(I)) < 4u)
#pragma unroll
                    for (int r = 0; r < 4; ++r) p[r] -= at == m_of(I) + r ? 1.f : 0.f;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    p[r] = counts ? p[r] * scale : 0.f;
                    over_n[I * 4 + r] += p[r] * power;
                }
                put_prob(I, p);
            }
            leave_prob(j);
        }
        if (g.bias_part || g.bias_out) {
            typedef typename ElementOf<P>::type E;
            const float factor = g.bias_out ? factor_of(g.factor) : 1.f;
            // Sums over the lanes of one m: with every exchange a lane keeps half of its words and sends the others' sums away,
            // until it has at most one word of its own (a fifth of the exchanges that summing all words in all lanes takes,
            // which cost 35 us of 146 for 1543 tokens and 20011 words).
            const int first = spread_sums<U::size / 2, MG * 4>(over_n, lane);
            constexpr int kOwn = MG * 4 > U::size ? MG * 4 / U::size : 1;
#pragma unroll
            for (int k = 0; k < kOwn; ++k) fl[wn * BM + m_in + m_of((first + k) / 4) + (first + k) % 4] = over_n[k];
            __syncthreads();
            for (int c = threadIdx.x; c < BM; c += WAVES * 64) {
                if (m0 + c >= g.M) continue;
                float s = fl[c];
#pragma unroll
                for (int w = 1; w < WN; ++w) s += fl[w * BM + c];
                if (g.bias_out) ((E *)g.bias_out)[m0 + c] = from_float<E>(s * factor);
                else g.bias_part[(int64_t)tn * g.ld_bias_part + m0 + c] = s;
            }
        }
    }
    if constexpr (KIND == kOut) {
        typedef typename ElementOf<P>::type E;
        const float all = g.slice ? 1.f : out_factor<P>(g.factor);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int own = n0 + n_in + j * U::size;
            const float factor = P::half && g.row_power && !g.slice && own < g.n_store ? all * g.row_power[own] : all;
            auto leave = [&](auto kind, int64_t ld, void *base) {
                typedef decltype(kind) S;
                typedef Gather<S, BM> Out;
#pragma unroll
                for (int I = 0; I < MG; ++I) {
                    const f32x4 v = f32x4{value(I, j, 0), value(I, j, 1), value(I, j, 2), value(I, j, 3)} * factor;
                    char *to = Out::at(lds, row_out, m_in + m_of(I));
                    if constexpr (sizeof(S) == 4) *(f32x4 *)to = v;
                    else *(s16x4 *)to = round4<P>(v);
                }
                __syncthreads();
                Out::template leave<kThreads>(lds, kRowsOut, g.M - m0, [&](int row) -> S * {
                    const int n = n0 + n_of(row, j);
                    return n < g.n_store ? (S *)base + n * ld + m0 : nullptr;
                });
                __syncthreads();
            };
            if (g.slice) leave(float{}, g.M, g.slice + (int64_t)split * g.n_store * g.M);
            else leave(E{}, g.ldo, g.out);
        }
    }
}

template <typename P, int BM, int BN, int WM, int WN, bool A_ACROSS, bool B_ACROSS, int KIND, int STAGES>
__global__ __launch_bounds__(WM * WN * 64) void product_kernel(Args g)
{
    __shared__ __attribute__((aligned(1024))) char lds[kLdsBytes<P, BM, BN, WM, WN, KIND, STAGES>];
    product_tile<P, BM, BN, WM, WN, A_ACROSS, B_ACROSS, KIND, STAGES>(g, blockIdx.x, lds);
}

// Of float32 weights as they are, for few tokens: logits (A along the reduction) and hidden gradients (across it).  Splitting a
// fragment into planes takes some 70 vector instructions, which run between the products of the one before; two workgroups
// on a CU cover each other's waits (37 tokens, 50021 words x 2048, the logits: 130 us; with five stages and one workgroup 200,
// with the split in one piece behind its loads 150; 410 MB of weights take 75).
template <int KIND, int WIDTH>
__global__ __launch_bounds__(256, 2) void raw_kernel(Args g)
{
    constexpr int BM = kRawWords, BN = kRawTokens, STAGES = 2;
    __shared__ __attribute__((aligned(1024))) char lds[kLdsBytes<Split, BM, BN, 4, 1, KIND, STAGES, true>];
    product_tile<Split, BM, BN, 4, 1, KIND == kOut, false, KIND, STAGES, WIDTH>(g, blockIdx.x, lds);
}

// Both gradients' products in one launch, `first` workgroups for the first.
template <typename P, int BM, int BN, int WM, int WN, int STAGES>
__global__ __launch_bounds__(WM * WN * 64) void both_kernel(Args hidden, Args weight, int first)
{
    __shared__ __attribute__((aligned(1024))) char lds[kLdsBytes<P, BM, BN, WM, WN, kOut, STAGES>];
    if ((int)blockIdx.x < first)
        product_tile<P, BM, BN, WM, WN, true, false, kOut, STAGES>(hidden, blockIdx.x, lds);
    else
        product_tile<P, BM, BN, WM, WN, true, true, kOut, STAGES>(weight, blockIdx.x - first, lds);
}

int launch_raw(int kind, int width, Args &g, hipStream_t st);

// Which product a launch is.
enum { kLogitStats = 0, kLogitKeep = 1, kLogitProb = 2, kHidden = 3, kWeight = 4 };

// Tile shapes, m x n, by their number in a launch.  For choosing among them: workgroups that a CU holds, and measured, in
// microseconds, a step of the reduction while every CU has its fill, a step while none has more than one workgroup, what a
// workgroup takes to begin and end, and what it takes besides where it leaves probabilities.
constexpr int kShapes = 4;
template <typename P> struct Shapes {
    static constexpr int m[kShapes] = {256, 128, 128, 64}, n[kShapes] = {256, 128, 64, 64}, resident[kShapes] = {1, 2, 2, 3};
    static constexpr float step_us[kShapes] = {1.6f, 1.05f, 0.8f, 0.5f}, alone_us[kShapes] = {1.0f, 0.6f, 0.5f, 0.3f};
    static constexpr float ends_us[kShapes] = {6.f, 8.f, 6.f, 4.f}, prob_us[kShapes] = {5.f, 10.f, 6.f, 3.f};
};
template <> struct Shapes<Split> {
    // the last for logits only
    static constexpr int m[kShapes] = {256, 128, 64, 32}, n[kShapes] = {128, 128, 64, 32}, resident[kShapes] = {1, 1, 1, 2};
    static constexpr float step_us[kShapes] = {2.5f, 1.6f, 0.75f, 0.5f}, alone_us[kShapes] = {2.0f, 1.1f, 0.57f, 0.38f};
    static constexpr float ends_us[kShapes] = {6.f, 5.f, 3.f, 3.f}, prob_us[kShapes] = {16.f, 8.f, 4.f, 3.f};
};
template <typename P> constexpr int kGradShapes = P::planes == 1 ? 4 : 3;

// Launches one product with tiles of shape `tile`; fills in the tile counts.  With `other` the two gradients' products run in
// one launch, both with that shape (g is kHidden, *other kWeight).  A translation unit per P.
template <typename P> int launch_product(int kind, int tile, Args &g, Args *other, hipStream_t st);

// The same for up to kFewTokens tokens of float32, with operands that lie as the caller's do (P excepted); the logits' tiles are
// kFewWords words of all tokens, hidden gradients always go to slices.
constexpr int kFewTokens = 16, kFewWords = 32;
int launch_few(int kind, int tokens, Args &g, hipStream_t st);

template <typename P, int BM, int BN, int WM, int WN, int STAGES, bool GRADS = true>
int launch_tiled(int kind, Args &g, Args *other, hipStream_t st)
{
    auto count = [](Args &x) {
        x.tiles_m = ceil_div(x.M, BM), x.tiles_n = ceil_div(x.N, BN);
        return (int64_t)x.tiles_m * x.tiles_n * x.splits;
    };
    const int64_t blocks = count(g), more = other ? count(*other) : 0;
    if (blocks + more > 0x7fffffff) return DS_ETOOLARGE;
    const dim3 grid((unsigned)(blocks + more)), threads(WM * WN * 64);
    if (kind == kLogitStats) {
        hipLaunchKernelGGL((product_kernel<P, BM, BN, WM, WN, false, false, kStats, STAGES>), grid, threads, 0, st, g);
    } else if (kind == kLogitKeep) {
        hipLaunchKernelGGL((product_kernel<P, BM, BN, WM, WN, false, false, kKeep, STAGES>), grid, threads, 0, st, g);
    } else if (kind == kLogitProb) {
        hipLaunchKernelGGL((product_kernel<P, BM, BN, WM, WN, false, false, kProb, STAGES>), grid, threads, 0, st, g);
    } else if constexpr (GRADS) {
        if (other)
            hipLaunchKernelGGL((both_kernel<P, BM, BN, WM, WN, STAGES>), grid, threads, 0, st, g, *other, (int)blocks);
        else if (kind == kHidden)
            hipLaunchKernelGGL((product_kernel<P, BM, BN, WM, WN, true, false, kOut, STAGES>), grid, threads, 0, st, g);
        else
            hipLaunchKernelGGL((product_kernel<P, BM, BN, WM, WN, true, true, kOut, STAGES>), grid, threads, 0, st, g);
    } else {
        return DS_EINVAL;
    }
    return launch_status();
}

}  // namespace vocab
}  // namespace ds
