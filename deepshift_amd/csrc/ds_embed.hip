// Embedding lookup with scaling, and its gradient by sorted tokens.
//
//   out[t][:] = scale * W[id_t][:]             dW[v][:] = scale * sum over { t : id_t = v, v != padding } of g[t][:]
//
// Both only move data.  The sum of a word's gradients runs over its tokens in ascending order, in 32 bits, and is rounded
// once: the tokens are sorted by word (stably), so no atomics touch the sums and a call repeats bit for bit.
#include "ds_train.h"

namespace ds {

// ---- lookup ------------------------------------------------------------------------------------------------

constexpr int kLookupUnits = 4;  // accesses a thread has in flight

// Bound by memory, and by the launch where there are few tokens.  A workgroup takes 256 * kLookupUnits consecutive accesses of
// the result, whatever the length of a row; row and column of its first one are the only 64-bit division.  The result passes
// the caches by, which leaves them to the rows that more tokens share: 131072 tokens of 4096 bfloat16 features from 131072
// words drawn as text has them take 320 us, 4.2 TB/s of what has to move (352 us with ordinary stores; 2 or 8 accesses a thread
// make no difference; a large copy reaches 4.9 TB/s).  64 tokens of 512: 3.4 us.
// ANY: rows that begin or end elsewhere than at multiples of 16 bytes; their accesses are as wide, the last one of a row but for
// what there is (65536 x 2047 bfloat16: 122 us, element by element 209, 77 for 2048).
template <typename E, bool ANY>
__global__ __launch_bounds__(256) void embed_kernel(const void *__restrict__ ids, int wide, const E *__restrict__ w,
                                                    E *__restrict__ out, int64_t T, int64_t V, int64_t D, int64_t ldw, float scale,
                                                    uint32_t per_row, FastDiv by_row)
{
    constexpr int N = 16 / sizeof(E);
    const uint64_t first = (uint64_t)blockIdx.x * (256 * kLookupUnits);
    const uint64_t row0 = first / per_row;
    const uint32_t rem0 = (uint32_t)(first - row0 * per_row);
    Vec<E, N> got[kLookupUnits];
    int id[kLookupUnits];
#pragma unroll
    for (int j = 0; j < kLookupUnits; ++j) {
        const uint32_t local = rem0 + j * 256 + threadIdx.x;
        const uint32_t r = div_by(local, by_row);
        const int64_t t = (int64_t)row0 + r;
        id[j] = t < T ? token_at(ids, wide, t, V) : -1;
        if (id[j] < 0) continue;
        const E *const row = w + (int64_t)id[j] * ldw;
        const uint32_t unit = local - r * per_row;
        if constexpr (ANY) got[j] = load_any<E, N>(row + (int64_t)unit * N, D - (int64_t)unit * N);
        else got[j] = ((const Vec<E, N> *)row)[unit];
    }
#pragma unroll
    for (int j = 0; j < kLookupUnits; ++j) {
        const uint64_t at = first + j * 256 + threadIdx.x;
        if (at >= (uint64_t)T * per_row) continue;
        Vec<E, N> o;
#pragma unroll
        for (int e = 0; e < N; ++e) o.v[e] = from_float<E>(id[j] >= 0 ? to_float(got[j].v[e]) * scale : NAN);
        if constexpr (ANY) {
            const uint32_t local = rem0 + j * 256 + threadIdx.x, r = div_by(local, by_row);
            const int64_t col = (int64_t)(local - r * per_row) * N;
            store_any<E, N>(out + ((int64_t)row0 + r) * D + col, o, D - col);
        } else {
            store_streaming((Vec<E, N> *)out + at, o);
        }
    }
}

template <typename E>
int launch_embed(const void *ids, int wide, const void *w, void *out, int64_t T, int64_t V, int64_t D, int64_t ldw,
                 float scale, hipStream_t st)
{
    constexpr int N = 16 / sizeof(E);
    const bool any = vector_elements(sizeof(E), {D, ldw}, {w, out}) < N;
    const uint64_t per_row = (uint64_t)((D + N - 1) / N), blocks = ((uint64_t)T * per_row + 256 * kLookupUnits - 1) / (256 * kLookupUnits);
    if (per_row > 0x7fffffffull - 256 * kLookupUnits || blocks > 0x7fffffffull) return DS_ETOOLARGE;
    const FastDiv by_row = fast_div((uint32_t)per_row);
    auto kernel = any ? embed_kernel<E, true> : embed_kernel<E, false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, st, ids, wide, (const E *)w, (E *)out, T, V, D, ldw, scale,
                       (uint32_t)per_row, by_row);
    return launch_status();
}

// ---- tokens sorted by word ------------------------------------------------------------------------------------

// The gradient begins as zeros, which words without tokens keep: most of a large table's.  Sorting takes a few CUs, so the
// launches that sort fill it besides, and rows with tokens are written once more.  (Filling empty rows alone, which took a
// launch that searches for them behind the sums: 8192 tokens of 2048 bfloat16 features, 131072 words, 139 us instead of 125; 500
// of 4096 float32 features 424, now 373; 131072 of 4096, 32768 words, most rows written twice, 425, now 389; 2065 of 385, 10007
// words, 24, now 20.)  They pass the caches by, which leaves those to the gradients.

// Zeros to a stretch of `bytes`, an even number, `units` times 16 bytes a thread.
struct Zeros {
    char *to;
    int64_t bytes;
    int units;
};
template <int THREADS>
__device__ __forceinline__ void fill_zeros(const Zeros &z, int block)
{
    const int64_t head = min(z.bytes, (int64_t)(-(uintptr_t)z.to & 15)), all = (z.bytes - head) >> 4, tail = head + (all << 4);
    Vec<uint32_t, 4> *const to = (Vec<uint32_t, 4> *)(z.to + head);
#pragma unroll 4
    for (int j = 0; j < z.units; ++j) {
        const int64_t u = ((int64_t)block * z.units + j) * THREADS + threadIdx.x;
        if (u < all) store_streaming(to + u, Vec<uint32_t, 4>{});
    }
    if (block > 0) return;
    if ((int)threadIdx.x * 2 < head) ((uint16_t *)z.to)[threadIdx.x] = 0;
    if ((int)threadIdx.x * 2 < z.bytes - tail) ((uint16_t *)(z.to + tail))[threadIdx.x] = 0;
}
// 16 KB a workgroup, up to 256 where all CUs have eight of them (2.1 GB: 438 us with 64 KB each, 386 with 128, 373 with 256).
inline Zeros zeros_of(void *to, int64_t bytes, int threads)
{
    const int64_t share = max((int64_t)16384, min((int64_t)262144, bytes / (8 * device_cus())));
    return Zeros{(char *)to, bytes, (int)(share / (threads * 16))};
}
inline int zero_blocks(const Zeros &z, int threads)
{
    const int64_t share = (int64_t)z.units * threads * 16;
    return (int)((z.bytes + share - 1) / share);
}

constexpr uint32_t kNoWord = 0xfffffffeu;  // sorts behind every word: padding, and what is no word at all

__device__ __forceinline__ uint32_t key_at(const void *ids, int wide, int64_t i, int64_t V, int64_t padding)
{
    const int id = token_at(ids, wide, i, V);
    return id < 0 || id == padding ? kNoWord : (uint32_t)id;
}

// Up to kRankMost tokens: the place of a token is the number of tokens with a smaller word, or the same word and an earlier
// position.  Every workgroup holds all words in LDS and places 64 tokens, its 16 waves each compare them with a sixteenth:
// T * T comparisons, two instructions each.  One launch: 7 us for 2065 tokens, 9 for 4096, 15 for 8192.  Against two of the passes
// below a whole gradient (of 128 features) takes 27 instead of 35 us for 9000 tokens, 31 and 37 for 12288, 36 and 33 for 16384;
// against one pass, which fewer than 511 words need, both take 22.7 for 6144 tokens, and that is half as many.
constexpr int kRankMost = 12288;  // a multiple of 128

// Workgroups behind those that sort fill `zeros` with zeros.
__global__ __launch_bounds__(1024) void embed_rank_kernel(const void *__restrict__ ids, int wide, int T, int64_t V,
                                                          int64_t padding, uint32_t *__restrict__ keys,
                                                          uint32_t *__restrict__ pos, Zeros zeros)
{
    __shared__ __attribute__((aligned(16))) uint32_t word[kRankMost];
    __shared__ uint32_t before[16][64];
    const int sorting = (T + 63) / 64;
    if ((int)blockIdx.x >= sorting) {
        fill_zeros<1024>(zeros, blockIdx.x - sorting);
        return;
    }
    const int padded = (T + 63) & ~63;
    for (int i = threadIdx.x; i < padded; i += 1024) word[i] = i < T ? key_at(ids, wide, i, V, padding) : kNoWord;
    __syncthreads();
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, t0 = blockIdx.x * 64;
    const uint32_t mine = word[t0 + lane];
    uint32_t n = 0;
    for (int g = wave * 64; g < padded; g += 16 * 64) {
        if (g == t0) {
            for (int i = 0; i < 64; ++i) n += word[g + i] < mine || (word[g + i] == mine && i < lane);
        } else {
            // of two equal words the earlier one comes first
            const uint32_t below = mine + (g < t0);
            const uint4 *four = (const uint4 *)(word + g);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const uint4 w = four[i];
                n += (w.x < below) + (w.y < below) + (w.z < below) + (w.w < below);
            }
        }
    }
    before[wave][lane] = n;
    __syncthreads();
    if (wave == 0 && t0 + lane < T) {
        uint32_t place = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) place += before[i][lane];
        keys[place] = mine;
        pos[place] = t0 + lane;
    }
}

// More tokens: a radix sort, least significant digit first, 9 bits a pass.  At most kSortBlocks workgroups, each with one
// stretch of the tokens; the counts of all of them (512 digits x 64) are few enough that every workgroup adds up its own
// offsets, so a pass is two launches.  Bound by their latency: 65536 tokens of 131072 words take two passes of 5 + 8.5 us.
constexpr int kDigitBits = 9, kDigits = 1 << kDigitBits, kSortBlocks = 64, kSortTile = 1024;

struct SortPass {
    const void *ids;  // first pass: the token numbers themselves; NULL later
    int wide;
    int64_t V, padding;
    const uint32_t *keys, *pos;
    uint32_t *out_keys, *out_pos;
    uint32_t *counts;  // [blocks][kDigits]
    int64_t T, stretch;
    int shift, blocks;  // workgroups from `blocks` on fill
    Zeros zeros;
};

__device__ __forceinline__ uint32_t sort_key(const SortPass &p, int64_t i)
{
    return p.ids ? key_at(p.ids, p.wide, i, p.V, p.padding) : p.keys[i];
}

__global__ __launch_bounds__(256) void embed_count_kernel(SortPass p)
{
    __shared__ uint32_t count[kDigits];
    if ((int)blockIdx.x >= p.blocks) {
        fill_zeros<256>(p.zeros, blockIdx.x - p.blocks);
        return;
    }
    for (int d = threadIdx.x; d < kDigits; d += 256) count[d] = 0;
    __syncthreads();
    const int64_t from = blockIdx.x * p.stretch, to = min(p.T, from + p.stretch);
    for (int64_t i = from + threadIdx.x; i < to; i += 256)
        atomicAdd(&count[(sort_key(p, i) >> p.shift) & (kDigits - 1)], 1u);  // whole numbers: any order gives the same
    __syncthreads();
    for (int d = threadIdx.x; d < kDigits; d += 256) p.counts[blockIdx.x * kDigits + d] = count[d];
}

__global__ __launch_bounds__(256) void embed_scatter_kernel(SortPass p)
{
    constexpr int kItems = kSortTile / 256;
    __shared__ uint32_t base[kDigits];      // where the next key of each digit goes
    __shared__ uint32_t seen[4][kDigits];   // keys of each digit that each wave has had in this tile
    __shared__ uint32_t wave_sum[4];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    if ((int)blockIdx.x >= p.blocks) {
        fill_zeros<256>(p.zeros, blockIdx.x - p.blocks);
        return;
    }
    {
        // two neighbouring digits a thread: totals, then an exclusive scan over the 512 digits
        uint32_t total[2] = {0, 0}, mine[2] = {0, 0};
        const uint2 *c = (const uint2 *)p.counts + threadIdx.x;
#pragma unroll 16
        for (int b = 0; b < p.blocks; ++b) {
            const uint2 v = c[b * (kDigits / 2)];
            total[0] += v.x, total[1] += v.y;
            if (b < (int)blockIdx.x) mine[0] += v.x, mine[1] += v.y;
        }
        const uint32_t own = total[0] + total[1];
        uint32_t run = own;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t up = __shfl_up(run, o);
            run += lane >= o ? up : 0;
        }
        if (lane == 63) wave_sum[wave] = run;
        __syncthreads();
        uint32_t front = run - own;
        for (int w = 0; w < wave; ++w) front += wave_sum[w];
        base[threadIdx.x * 2] = front + mine[0];
        base[threadIdx.x * 2 + 1] = front + total[0] + mine[1];
    }
    const int64_t from = blockIdx.x * p.stretch, to = min(p.T, from + p.stretch);
    for (int64_t tile = from; tile < to; tile += kSortTile) {
        for (int i = threadIdx.x; i < 4 * kDigits; i += 256) (&seen[0][0])[i] = 0;
        __syncthreads();
        // a wave has a contiguous quarter of the tile, 64 keys at a time
        uint32_t key[kItems], at[kItems], rank[kItems];
#pragma unroll
        for (int j = 0; j < kItems; ++j) {
            const int64_t i = tile + wave * (kSortTile / 4) + j * 64 + lane;
            const bool valid = i < to;
            key[j] = valid ? sort_key(p, i) : kNoWord;
            at[j] = valid ? (p.ids ? (uint32_t)i : p.pos[i]) : 0;
            const uint32_t digit = (key[j] >> p.shift) & (kDigits - 1);
            // the lanes that hold the same digit, counting only real keys
            uint64_t same = __ballot(valid);
#pragma unroll
            for (int b = 0; b < kDigitBits; ++b) {
                const uint64_t set = __ballot((digit >> b) & 1);
                same &= (digit >> b) & 1 ? set : ~set;
            }
            const uint32_t earlier = seen[wave][digit];  // one wave, program order: read by all before the first lane adds
            __builtin_amdgcn_wave_barrier();
            const uint32_t lower = __popcll(same & ((1ull << lane) - 1));
            rank[j] = earlier + lower;
            if (valid && lower == 0) seen[wave][digit] = earlier + (uint32_t)__popcll(same);
            __builtin_amdgcn_wave_barrier();
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kItems; ++j) {
            const int64_t i = tile + wave * (kSortTile / 4) + j * 64 + lane;
            if (i >= to) continue;
            const uint32_t digit = (key[j] >> p.shift) & (kDigits - 1);
            uint32_t place = base[digit] + rank[j];
            for (int w = 0; w < wave; ++w) place += seen[w][digit];
            p.out_keys[place] = key[j];
            p.out_pos[place] = at[j];
        }
        __syncthreads();
        for (int d = threadIdx.x; d < kDigits; d += 256) base[d] += seen[0][d] + seen[1][d] + seen[2][d] + seen[3][d];
        __syncthreads();
    }
}

// ---- sums ------------------------------------------------------------------------------------------------------

// The sorted tokens are cut into chunks; a wave adds up one chunk for 64 * N columns.  A word whose tokens lie in one chunk
// is finished there.  One that runs on leaves a partial sum: in slot 1 of the chunk that it begins in, in slot 0 of the
// others; embed_join_kernel joins them in order, so that a word with most of the tokens does not wait for one wave.  Bound by
// memory: 65536 x 2048 bfloat16 gradients of words drawn evenly in, 0.27 GB, and 0.21 GB of finished rows out in 90 us.  Eight
// rows are on their way at a time; sixteen take more registers than they hide (151 us where eight took 114).
template <typename E, int N, bool ANY>
__global__ __launch_bounds__(64) void embed_sum_kernel(const E *__restrict__ g, int64_t ldg, const uint32_t *__restrict__ keys,
                                                       const uint32_t *__restrict__ pos, E *__restrict__ dw,
                                                       float *__restrict__ part, int64_t T, int64_t D, int chunk, float scale)
{
    const int64_t from = (int64_t)blockIdx.x * chunk, to = min(T, from + chunk);
    const int64_t col = ((int64_t)blockIdx.y * 64 + threadIdx.x) * N;
    const bool in = col < D;
    const int left = (int)min(D - col, (int64_t)N);
    const uint32_t before = from > 0 ? keys[from - 1] : kNoWord;
    const uint32_t behind = to < T ? keys[to] : kNoWord;
    float acc[N];
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = 0.f;
    uint32_t run = keys[from];
    bool first = true;
    constexpr int kAhead = 8;  // rows on their way
    for (int64_t i = from; i < to; i += kAhead) {
        Vec<E, N> got[kAhead];
        uint32_t key[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const bool real = i + j < to;
            key[j] = real ? keys[i + j] : kNoWord;
            if (real && key[j] != kNoWord && in) {
                const E *const row = g + (int64_t)pos[i + j] * ldg + col;
                if constexpr (ANY) got[j] = load_any<E, N>(row, left);
                else got[j] = *(const Vec<E, N> *)row;
            }
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            if (i + j >= to) break;
            if (key[j] != run) {
                // the run ends inside this chunk
                if (run != kNoWord && in) {
                    if (first && run == before) {
#pragma unroll
                        for (int e = 0; e < N; ++e)
                            if (!ANY || e < left) part[(int64_t)blockIdx.x * 2 * D + col + e] = acc[e];
                    } else {
                        Vec<E, N> o;
#pragma unroll
                        for (int e = 0; e < N; ++e) o.v[e] = from_float<E>(acc[e] * scale);
                        if constexpr (ANY) store_any<E, N>(dw + (int64_t)run * D + col, o, left);
                        else store_streaming((Vec<E, N> *)(dw + (int64_t)run * D + col), o);
                    }
                }
                first = false;
                run = key[j];
#pragma unroll
                for (int e = 0; e < N; ++e) acc[e] = 0.f;
            }
            if (run == kNoWord || !in) continue;
#pragma unroll
            for (int e = 0; e < N; ++e) acc[e] += to_float(got[j].v[e]);
        }
    }
    if (run == kNoWord || !in) return;
    const bool came = first && run == before, goes = run == behind;
    if (came || goes) {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (!ANY || e < left) part[((int64_t)blockIdx.x * 2 + (came ? 0 : 1)) * D + col + e] = acc[e];
    } else {
        Vec<E, N> o;
#pragma unroll
        for (int e = 0; e < N; ++e) o.v[e] = from_float<E>(acc[e] * scale);
        if constexpr (ANY) store_any<E, N>(dw + (int64_t)run * D + col, o, left);
        else store_streaming((Vec<E, N> *)(dw + (int64_t)run * D + col), o);
    }
}

// The first of `n` sorted keys that is not below v, found by a whole wave: 64 probes a round.
__device__ __forceinline__ uint32_t wave_lower_bound(const uint32_t *__restrict__ keys, uint32_t n, uint32_t v)
{
    uint32_t lo = 0, left = n;  // the answer is in [lo, lo + left]
    while (left > 0) {
        const uint32_t stride = (left + 63) / 64, at = (threadIdx.x & 63) * stride;
        const bool below = at < left && keys[lo + at] < v;
        const uint32_t passed = (uint32_t)__popcll(__ballot(below));
        if (passed == 0) break;
        // keys[lo + (passed - 1) * stride] is below v, the next probe is not
        const uint32_t skip = (passed - 1) * stride + 1;
        const uint32_t end = passed * stride < left ? passed * stride : left;
        lo += skip, left = end - skip;
    }
    return lo;
}

// The partial sums of a word that begins in chunk c0 and ends in c1, in order; `p` is chunk 0's slot 0, at the columns wanted.
template <typename E, int N, bool ANY>
__device__ __forceinline__ Vec<E, N> joined(const float *__restrict__ p, uint32_t c0, uint32_t c1, int64_t D, int left, float scale)
{
    float acc[N];
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = !ANY || e < left ? p[((int64_t)c0 * 2 + 1) * D + e] : 0.f;
    constexpr int kAhead = N <= 2 ? 24 : 8;  // partial sums on their way
    for (uint32_t c = c0 + 1; c <= c1; c += kAhead) {
        Vec<float, N> got[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            if (c + j > c1) continue;
            const float *const at = p + (int64_t)(c + j) * 2 * D;
            if constexpr (ANY) got[j] = load_any<float, N>(at, left);
            else got[j] = *(const Vec<float, N> *)at;
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
#pragma unroll
            for (int e = 0; e < N; ++e) acc[e] += c + j <= c1 ? got[j].v[e] : 0.f;
    }
    Vec<E, N> o;
#pragma unroll
    for (int e = 0; e < N; ++e) o.v[e] = from_float<E>(acc[e] * scale);
    return o;
}

// Words in several chunks: their joined sums, by the workgroup of the chunk that such a word begins in.  Bound by latency: 44
// partial sums of the most frequent of 2065 tokens in 4.4 us.
template <typename E, int N, bool ANY>
__global__ __launch_bounds__(64) void embed_join_kernel(const uint32_t *__restrict__ keys, const float *__restrict__ part,
                                                        E *__restrict__ dw, int64_t T, int64_t D, int chunk, float scale)
{
    const int64_t from = (int64_t)blockIdx.x * chunk, to = min(T, from + chunk);
    if (to >= T) return;
    const uint32_t run = keys[to - 1];
    if (run == kNoWord || keys[to] != run || (from > 0 && keys[from - 1] == run)) return;
    const uint32_t end = (uint32_t)to + wave_lower_bound(keys + to, (uint32_t)(T - to), run + 1);
    const int64_t col = ((int64_t)blockIdx.y * 64 + threadIdx.x) * N;
    if (col >= D) return;
    const int left = (int)min(D - col, (int64_t)N);
    const Vec<E, N> o = joined<E, N, ANY>(part + col, blockIdx.x, (end - 1) / chunk, D, left, scale);
    if constexpr (ANY) store_any<E, N>(dw + (int64_t)run * D + col, o, left);
    else *(Vec<E, N> *)(dw + (int64_t)run * D + col) = o;
}

// Tokens a chunk: long ones leave hot words fewer partial sums to join, short ones more waves (2065 tokens, 700 of them one word:
// 5 us to add up and 12 to join with 16 a chunk, 9 and 9.5 with 32).
inline int embed_chunk(int64_t T) { return T <= 4096 ? 16 : T <= 32768 ? 32 : T <= 131072 ? 64 : 128; }

struct EmbedSpace {
    size_t keys[2], pos[2], counts, part, bytes;
};
inline EmbedSpace embed_space(int64_t T, int64_t D)
{
    EmbedSpace s;
    const size_t list = align_up((size_t)T * 4, 256);
    size_t at = 0;
    for (int i = 0; i < 2; ++i) {
        s.keys[i] = at, at += list;
        s.pos[i] = at, at += list;
    }
    s.counts = at, at += (size_t)kDigits * kSortBlocks * 4;
    const int64_t chunks = (T + embed_chunk(T) - 1) / embed_chunk(T);
    s.part = at, at += align_up((size_t)chunks * 2 * (size_t)D * 4, 256);
    s.bytes = at;
    return s;
}

// How the sums' launches go over a gradient: `width` columns a lane, `any`: wherever its rows begin.
struct SumGrid {
    int width, chunk;
    bool any;
    int64_t chunks, slices;
    bool fits() const { return chunks <= 0x7fffffff && slices <= 65535; }
};
inline SumGrid sum_grid(int bytes, const void *g, int64_t ldg, const void *dw, int64_t T, int64_t D)
{
    const int wide = 16 / bytes;
    SumGrid s{vector_elements(bytes, {D, ldg}, {g, dw}), embed_chunk(T), false, 0, 0};
    s.chunks = (T + s.chunk - 1) / s.chunk;
    auto slices_of = [&](int width) { return ((D + width - 1) / width + 63) / 64; };
    // Rows that allow one element at a time: as wide as others, wherever they begin, where that leaves every CU four waves
    // (65536 x 2047 bfloat16 282, now 199 us, x 1023 float32 171 and 145; but 2065 x 385 float32 17 us, and 24 that way).
    s.any = s.width == 1 && s.chunks * slices_of(wide) >= 4 * device_cus();
    if (s.any) s.width = wide;
    s.slices = slices_of(s.width);
    return s;
}

template <typename E>
int launch_embed_grad(const SumGrid &s, const uint32_t *keys, const uint32_t *pos, const void *g, int64_t ldg, void *dw, float *part,
                      int64_t T, int64_t D, float scale, hipStream_t st)
{
    constexpr int kWide = 16 / sizeof(E);
    const int n = s.width, chunk = s.chunk;
    const bool any = s.any;
    const dim3 grid((unsigned)s.chunks, (unsigned)s.slices);
#define DS_LAUNCH(N, ANY)                                                                                                 \
    do {                                                                                                                  \
        hipLaunchKernelGGL((embed_sum_kernel<E, N, ANY>), grid, dim3(64), 0, st, (const E *)g, ldg, keys, pos, (E *)dw, part, T, \
                           D, chunk, scale);                                                                              \
        hipLaunchKernelGGL((embed_join_kernel<E, N, ANY>), grid, dim3(64), 0, st, keys, part, (E *)dw, T, D, chunk, scale); \
    } while (0)
    if (any) DS_LAUNCH(kWide, true);
    else if (n == 8) { if constexpr (sizeof(E) == 2) DS_LAUNCH(8, false); }
    else if (n == 4) DS_LAUNCH(4, false);
    else if (n == 2) DS_LAUNCH(2, false);
    else DS_LAUNCH(1, false);
#undef DS_LAUNCH
    return launch_status();
}

// The tokens in order of their words; the launches on the way also fill `bytes` at `zeros` with zeros.
int sort_tokens(const void *ids, int wide, int64_t T, int64_t V, int64_t padding, char *ws, const EmbedSpace &s, void *zeros,
                int64_t bytes, hipStream_t st, const uint32_t **keys, const uint32_t **pos)
{
    uint32_t *k[2] = {(uint32_t *)(ws + s.keys[0]), (uint32_t *)(ws + s.keys[1])};
    uint32_t *p[2] = {(uint32_t *)(ws + s.pos[0]), (uint32_t *)(ws + s.pos[1])};
    int at = 0;
    // the low bits of kNoWord, all set but the last, have to stay above every word
    int bits = 1;
    while (((int64_t)1 << bits) <= V + 1) ++bits;
    if (T == 0 || (T <= (bits > kDigitBits ? kRankMost : kRankMost / 2) && g_tune.embed_radix != 1)) {
        const Zeros z = zeros_of(zeros, bytes, 1024);
        hipLaunchKernelGGL(embed_rank_kernel, dim3((unsigned)((T + 63) / 64 + zero_blocks(z, 1024))), dim3(1024), 0, st, ids, wide,
                           (int)T, V, padding, k[0], p[0], z);
    } else {
        int64_t blocks = min((int64_t)kSortBlocks, (T + kSortTile - 1) / kSortTile);
        const int64_t stretch = ((T + blocks - 1) / blocks + kSortTile - 1) / kSortTile * kSortTile;
        blocks = (T + stretch - 1) / stretch;
        // every launch fills its share
        const int launches = (bits + kDigitBits - 1) / kDigitBits * 2;
        const int64_t share = (bytes / launches / 65536 + 1) * 65536;
        int64_t filled = 0;
        SortPass pass{ids, wide, V, padding, nullptr, nullptr, k[0], p[0], (uint32_t *)(ws + s.counts), T, stretch, 0, (int)blocks, {}};
        for (int shift = 0; shift < bits; shift += kDigitBits) {
            pass.shift = shift;
            if (shift > 0) {
                pass.ids = nullptr;
                pass.keys = k[at], pass.pos = p[at];
                at ^= 1;
                pass.out_keys = k[at], pass.out_pos = p[at];
            }
            for (auto kernel : {embed_count_kernel, embed_scatter_kernel}) {
                const int64_t now = min(share, bytes - filled);
                pass.zeros = zeros_of((char *)zeros + filled, now, 256);
                filled += now;
                hipLaunchKernelGGL(kernel, dim3((unsigned)(blocks + zero_blocks(pass.zeros, 256))), dim3(256), 0, st, pass);
            }
        }
    }
    *keys = k[at], *pos = p[at];
    return launch_status();
}

}  // namespace ds

using namespace ds;

DS_EXPORT int ds_embed(const void *ids, int id_bytes, const void *weight, int64_t ldw, void *out, int64_t T, int64_t V,
                       int64_t D, float scale, int type, ds_stream_t stream)
{
    if (T < 0 || V < 0 || D < 0 || !element_bytes(type) || (id_bytes != 4 && id_bytes != 8)) return DS_EINVAL;
    if (T == 0 || D == 0) return DS_OK;
    if (!ids || !out || (V > 0 && (!weight || ldw < D))) return DS_EINVAL;
    if (V > 0x7fffffff || T > 0x7fffffff) return DS_ETOOLARGE;
    const int wide = id_bytes == 8;
    hipStream_t st = (hipStream_t)stream;
    if (type == DS_F32) return launch_embed<float>(ids, wide, weight, out, T, V, D, ldw, scale, st);
    if (type == DS_BF16) return launch_embed<bf16_t>(ids, wide, weight, out, T, V, D, ldw, scale, st);
    return launch_embed<f16_t>(ids, wide, weight, out, T, V, D, ldw, scale, st);
}

DS_EXPORT size_t ds_embed_grad_workspace_bytes(int64_t T, int64_t D)
{
    return T < 0 || D < 0 ? 0 : embed_space(T, D).bytes;
}

DS_EXPORT int ds_embed_grad(const void *ids, int id_bytes, const void *grad, int64_t ldg, void *dweight, int64_t T, int64_t V,
                            int64_t D, int64_t padding, float scale, int type, void *workspace, size_t workspace_bytes,
                            ds_stream_t stream)
{
    if (T < 0 || V < 0 || D < 0 || !element_bytes(type) || (id_bytes != 4 && id_bytes != 8)) return DS_EINVAL;
    if (V == 0 || D == 0) return DS_OK;
    if (!dweight || (T > 0 && (!ids || !grad || ldg < D))) return DS_EINVAL;
    if (V > 0x7fffffff || T > 0x7fffffff || D > 0x7fffffff || V * D > (int64_t)1 << 44) return DS_ETOOLARGE;
    const SumGrid sums = sum_grid(element_bytes(type), grad, ldg, dweight, T, D);
    if (T > 0 && !sums.fits()) return DS_ETOOLARGE;
    const EmbedSpace s = embed_space(T, D);
    if (workspace_bytes < s.bytes || !workspace || (uintptr_t)workspace % 16) return DS_EWORKSPACE;
    hipStream_t st = (hipStream_t)stream;
    const uint32_t *keys, *pos;
    const int64_t bytes = V * D * (int64_t)element_bytes(type);
    const int status = sort_tokens(ids, id_bytes == 8, T, V, padding, (char *)workspace, s, dweight, bytes, st, &keys,
                                   &pos);
    if (status != DS_OK || T == 0) return status;
    float *part = (float *)((char *)workspace + s.part);
    if (type == DS_F32) return launch_embed_grad<float>(sums, keys, pos, grad, ldg, dweight, part, T, D, scale, st);
    if (type == DS_BF16) return launch_embed_grad<bf16_t>(sums, keys, pos, grad, ldg, dweight, part, T, D, scale, st);
    return launch_embed_grad<f16_t>(sums, keys, pos, grad, ldg, dweight, part, T, D, scale, st);
}
