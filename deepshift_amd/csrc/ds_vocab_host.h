// What the host's sides of the products of ds_vocab.h share: operands as the products take them, the choice of their tiles, and the
// joins of their slices.
#pragma once
#include "ds_vocab.h"
#include <algorithm>

namespace ds {
namespace vocab {

#define DS_TRY(what)                    \
    do {                                \
        const int s_ = (what);          \
        if (s_ != DS_OK) return s_;     \
    } while (0)

// An operand on its way to rows of Dp elements (pack_kernel in ds_vocab.hip).
struct Pack {
    const void *x;
    int64_t ld, rows;
    int D, Dp;
    uint16_t *out;
    int64_t ldo;
    const void *target;
    int wide;
    int64_t ignore;
    int64_t again;   // of 16 bits: rows are written once more, so many rows behind; or 0
};
// One operand, or two in one launch.  For float, bf16_t and f16_t.
template <typename E> int launch_pack(const Pack &one, const Pack &two, hipStream_t st);

// The sums of a bias's tiles, to the gradient of its words.
struct BiasJoin {
    const float *part;
    int ld, tiles, n;
    void *out;
};
// For float, bf16_t and f16_t.
template <typename E> int launch_bias_join(const BiasJoin &b, const float *f0, const float *f1, hipStream_t st);

// The slices of a product to `count` results in rows of M, packed, times the factors.
template <typename P> int launch_join(const float *slices, int splits, int64_t count, int M, const float *f0, const float *f1, void *out,
                                      hipStream_t st);

inline bool in_place(const void *p, int64_t ld, int64_t D) { return (uintptr_t)p % 16 == 0 && ld % 8 == 0 && D % 8 == 0; }

// What a call does: the loss, the gradients, or both.
enum { kLoss = 1, kGrad = 2 };

// Up to how many tokens of float32 read the weights as they are.  Small heads give each workgroup too little to read: 16 tokens of
// 512 features, 1000 words, 44 us a step where planes take 33 (8 tokens: 31 and 34), 16 of 1024, 8000 words, 74 and 78.
constexpr int64_t kManyWeights = 1 << 23;
inline int64_t few_tokens(int64_t weights) { return weights < kManyWeights ? kFewTokens / 2 : kFewTokens; }

// Up to how many tokens of float32 the matrix instructions take weights as they are, `width` floats at a time, split into planes by
// every tile of 64 tokens; for more, planes for all of them to share are worth what writing and reading them takes, the sooner the
// fewer weights there are, for gradients (whose hidden states are in planes either way) and for weights that come one by one.
// Measured as they are and by planes, in us:
//                                  loss of 24       128         512     a step of 24         128           256           512 tokens
//   1024 features,  8200 words      46   44     47   62     93   94      93   88    117  121     166  152       260  225
//   1024,          16400            45   69     61   72    140  153     108  137    163  169     252  265       412  412
//   1024,          33000            60  126     93  154    243  271     158  242    267  330     424  482       735  753
//   1023 (one by one), 8300         53   42     55   60    106   94     105   88    131  123     180  155       285  228
//   1023,          16400            54   70     67   73    158  153     120  138    176  171     276  267       451  415
//   1023,          33000            66  132    106  159    268  274     174  251    294  338     464  490       805  760
//   2049,          50021           143  389    242  410    767  796     437  706    737  898    1266 1332      2424 2206
constexpr int64_t kManyOddWeights = 7 << 21;
inline int64_t raw_tokens(int64_t weights, int width, int what)
{
    const bool odd = width == 1, grad = what & kGrad;
    if (weights < (odd ? kManyOddWeights : kManyWeights)) return 0;
    return std::min<int64_t>(odd && grad ? 256 : 512, weights >> (15 + odd + grad));
}

// The tile shape of a product, and how many stretches its reduction of k is cut into (1 of `most_splits`): the pair with the
// shortest estimate, rounds of workgroups times their steps and ends; slices are written and read once more by a launch of
// their own.  What decides it, measured: hidden gradients of 1543 x 1000 from 20011 words, float16, 157 us on 128 x 128 tiles
// in two stretches, 76 us on 256 x 256 in eight; 2048 x 1024 from 32768 words, float32, 1113 us (128 x 128, two) and 707 us
// (256 x 128, four); 64 x 512 from 1000 words, float32, 25 us in one stretch, 13 in four; scores of 512 tokens of 1024 features
// over 8000 words, bfloat16, 25, 16, 16 and 19 us from the largest tiles to the smallest.
struct Choice { int tile, splits; };
template <typename P>
Choice choose(int64_t m, int64_t n, int64_t k, int shapes, int most_splits, bool prob)
{
    typedef Shapes<P> S;
    const int cus = device_cus(), tile_knob = g_tune.vocab_tile, split_knob = g_tune.vocab_split;
    const int64_t steps = (k + P::step - 1) / P::step;
    Choice best{0, 1};
    if (m < 1 || n < 1) return best;
    double shortest = 1e300;
    for (int i = 0; i < shapes; ++i) {
        if (tile_knob >= 0 && tile_knob < shapes && i != tile_knob) continue;
        const int64_t tiles = ((m + S::m[i] - 1) / S::m[i]) * ((n + S::n[i] - 1) / S::n[i]);
        const int64_t fill = (int64_t)cus * S::resident[i];
        // stretches of 256 at least, and no more workgroups than two rounds of them
        int most = most_splits;
        if (most > steps * P::step / 256) most = (int)(steps * P::step / 256);
        if (split_knob >= 1) most = most < split_knob ? most : split_knob;
        else if (most > 2 * fill / tiles) most = (int)(2 * fill / tiles);
        if (most < 1) most = 1;
        for (int s = split_knob >= 1 ? most : 1; s <= most; s += 1 + s / 4) {
            const int64_t blocks = tiles * s;
            const double step = blocks <= cus ? S::alone_us[i] : S::step_us[i];
            const double round = (double)((steps + s - 1) / s) * step + S::ends_us[i] + (prob ? S::prob_us[i] : 0);
            const double us = (double)((blocks + fill - 1) / fill) * round + (s > 1 ? 4 + (double)s * m * n * 4 / 3e6 : 0);
            if (us < shortest) shortest = us, best = Choice{i, s};
        }
    }
    return best;
}

}  // namespace vocab
}  // namespace ds
