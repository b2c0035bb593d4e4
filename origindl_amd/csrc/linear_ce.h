// What the two implementations of the output layer with its loss share: linear_ce.hip (many rows) and linear_ce_rows.hip (few).
#pragma once
#include <cmath>

#include "odl_common.h"

namespace odl
{
namespace linear_ce
{
constexpr int kBlock = 256;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kDScale = 32768.f;  // d lies in [-1, 1]: two float16 numbers keep 2^-22 of an element, or 2^-40

// saved[] — what the forward pass leaves for the backward pass and the caller
enum Saved
{
    kLoss = 0,     // mean loss over the counted rows
    kBadLabel,     // int: a label outside [0, V) that is not ignore_index
    kCounted,      // rows that count
    kScaleX,       // the powers of two the operands were multiplied by
    kScaleW,
    kTicket,       // int: workgroups of the joining launch that are done
    kSavedWords = 8
};

__device__ inline int64_t label_of(const void *t, int is64, int64_t n)
{
    return is64 ? static_cast<const int64_t *>(t)[n] : (int64_t) static_cast<const int32_t *>(t)[n];
}

struct Labels
{
    const void *t;
    int is64;
    int64_t ignore, V, N;
    // the row's label, or -1 where the row does not count (ignored, out of range, or past the batch)
    __device__ int64_t operator()(int64_t n) const
    {
        if (n >= N)
            return -1;
        const int64_t l = label_of(t, is64, n);
        return l == ignore || l < 0 || l >= V ? -1 : l;
    }
};

// 2^v, one instruction (1 unit in the last place; results under 2^-126 are 0)
__device__ inline float pow2(float v)
{
    return __builtin_amdgcn_exp2f(v);
}

// e^(z - m). The difference first: a logit times log2(e) overflows from 2.4e38 on, and a mask may hold the type's lowest value.
__device__ inline float exp_under(float z, float m)
{
    return pow2((z - m) * kLog2e);
}

// what is subtracted from logits whose maximum is m: with m = -inf (an empty set, or logits that are all -inf) nothing, and the
// powers are 0
__device__ inline float finite_top(float m)
{
    return m == -INFINITY ? 0.f : m;
}

// merges (maximum m, s = sum e^(z - m)) of two sets of logits. fmaxf drops NaN from the maxima, the sums keep it. S: float within a tile, double over
// the tiles, of which a large vocabulary has millions
template <class S>
__device__ inline void merge(float &m, S &s, float m_o, S s_o)
{
    const float top = fmaxf(m, m_o), sub = finite_top(top);
    s = s * (S)exp_under(m, sub) + s_o * (S)exp_under(m_o, sub);
    m = top;
}

inline size_t aligned(size_t n)
{
    return (n + 255) & ~(size_t)255;
}

struct Carver
{
    char *at;
    size_t used = 0;
    template <class U>
    U *take(size_t bytes)
    {
        U *p = reinterpret_cast<U *>(at ? at + used : nullptr);
        used += aligned(bytes);
        return p;
    }
};


struct Problem
{
    const float *x, *w, *b;
    int w_out_in;
    Labels labels;
    int64_t N, K, V;
};

// Few rows over large weights: the bytes of the weights are what a pass costs, and they are read as they lie, no operand laid out
// first. Measured in us, weights [K, V], streams against operands laid out: one row over 2048 x 32000, forward, 61 and 231;
// forward and backward over 2048 x 100000 64 rows 877 and 1930, 128 rows 1343 and 2232, 256 rows 2314 and 2570. A tile of the
// streams holds 32, 64 or 128 rows, and a part of one costs the whole: under 6 million weights operands laid out win from 65 rows
// on (1024 x 4000: 80 rows 94 and 86, 256 rows 113 and 95; up to 64 rows the streams are up to a quarter faster there as well).
// The rule does not look at the weights' shape. Narrow ones, which d outweighs, would be faster laid out from 65 rows on (64 x 128000:
// 128 rows 331 and 176, 64 rows 178 and 161; 256 x 32000: 128 rows 154 and 114), and so would short vocabularies, whose few tiles
// leave compute units idle (7000 x 900: 128 rows 215 and 189).
inline bool few_rows(int64_t N, int64_t K, int64_t V)
{
    return N <= 256 && K * V >= 6000000;
}
size_t few_kept_floats(int64_t N, int64_t K, int64_t V);  // of logits that stay behind the row statistics
size_t few_forward_bytes(int64_t N, int64_t K, int64_t V);
size_t few_backward_bytes(int64_t N, int64_t K, int64_t V);
int few_forward(const Problem &p, float *saved, float *row_stats, char *workspace, hipStream_t st);
int few_backward(const Problem &p, const float *gy, const float *saved, const float *row_stats, float *gx, float *gw, float *gb, char *workspace,
                 hipStream_t st);
// the partial maxima and sums [tiles][n_pad] joined: row statistics, loss, flag and count; saved's ticket must be 0
int join(const float *part_m, const float *part_s, const float *target, int64_t tiles, int64_t n_pad, const Labels &labels, float *row_stats, void *scratch,
         float *saved, hipStream_t st);
size_t join_scratch_bytes(int64_t N);
}  // namespace linear_ce
}  // namespace odl
