// The output layer with its loss for up to 256 rows over large weights: scoring a few positions, small batches.
//
// What bounds it: the bytes of w. So nothing is laid out first: w streams once from where it lies through the registers into
// the matrix instructions, per pass:
//   forward    one pass: logits of 128 (64) entries a workgroup, their maximum and sum of powers in its epilogue
//   backward   the logits, which the forward pass has kept if they are small beside the weights (else one pass for them again):
//              the same epilogue in both cases writes d = softmax - one-hot (the weights' size times 3N / K) and gb; one pass for
//              gx = d.w, in runs of the vocabulary; gw = d^T.x writes its size once. d takes 12 bytes a row and entry: beyond
//              512 MB of it the vocabulary goes through in pieces, whose sums for gx add up.
//
// Mathematics. A float32 number is the sum of three bfloat16 numbers, its first, second and third eight bits, cut off without
// rounding: exact (elements under 2^-110 to 2^-133, bfloat16's smallest number). Of the nine products of two such sums the six of
// at least 2^-16 of the whole are formed by bfloat16 matrix instructions (v_mfma_f32_32x32x16_bf16), exact in float32, and summed
// there: what is left out is under 2^-23 of |a||b|. No scale is needed, as bfloat16 has float32's exponents, and so no pass over w
// to find one. Six products take 0.38 of the float32 matrix instruction's time. Measured: one row over 2048 x 32000, weights
// [K, V], the forward pass streams 262 MB in 47 to 52 us (5.0 to 5.5 TB/s; a copy of 4 GiB reaches 4.8); over 2048 x 100000, [K, V] and
// [V, K], forward and backward, 8 rows 700 and 735 us, 64 rows 877 and 895, 128 rows 1343 and 1360, 256 rows 2314 and 2350: past
// 64 rows the splitting and the products take longer than the bytes.
//
// Both products with w are one kernel: w is [out][contraction] for the logits of a [V, K] weight and [contraction][out] for its
// gx, and the other way round for a [K, V] weight. Eight waves share a tile of outputs, each takes an eighth of the contraction,
// 16 values a step, splits what it read and multiplies it with the small operand (x or d), which lies split, in the order of
// the instructions' lanes.
#include <algorithm>

#include "linear_ce.h"

namespace
{
using namespace odl::linear_ce;
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kWaves = 8;
constexpr int kFragment = 3 * 64;  // u32x4 of a block of 32 rows x 16 contraction values: three parts, 16 bytes a lane

// eight float32 into their first, second and third eight bits
__device__ inline void split3(const float *v, u32x4 *part)
{
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        const float a0 = v[2 * i], b0 = v[2 * i + 1];
        const unsigned a = __float_as_uint(a0), b = __float_as_uint(b0);
        const float a1 = a0 - __uint_as_float(a & 0xffff0000u), b1 = b0 - __uint_as_float(b & 0xffff0000u);
        const unsigned am = __float_as_uint(a1), bm = __float_as_uint(b1);
        const float a2 = a1 - __uint_as_float(am & 0xffff0000u), b2 = b1 - __uint_as_float(bm & 0xffff0000u);
        // the upper halves of both, the first value in the lower half
        part[0][i] = __builtin_amdgcn_perm(b, a, 0x07060302u);
        part[1][i] = __builtin_amdgcn_perm(bm, am, 0x07060302u);
        part[2][i] = __builtin_amdgcn_perm(__float_as_uint(b2), __float_as_uint(a2), 0x07060302u);
    }
}

__device__ inline f32x16 mfma(const u32x4 &a, const u32x4 &b, const f32x16 &c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// c += a . b: the small products first
__device__ inline void multiply(f32x16 &c, const u32x4 *a, const u32x4 *b)
{
    c = mfma(a[0], b[2], c);
    c = mfma(a[2], b[0], c);
    c = mfma(a[1], b[1], c);
    c = mfma(a[0], b[1], c);
    c = mfma(a[1], b[0], c);
    c = mfma(a[0], b[0], c);
}

__device__ inline void store3(u32x4 *at, const float *v, int lane)
{
    u32x4 part[3];
    split3(v, part);
#pragma unroll
    for (int p = 0; p < 3; ++p)
        at[p * 64 + lane] = part[p];
}

// x split: by_n as the small operand of the logits, [K / 16][blocks of 32 rows]; by_k as an operand of gw, rows of K, [K / 32][rows
// / 16] (null: not wanted). A wave makes one fragment of each. Also clears the ticket of the joining launch.
__global__ __launch_bounds__(kBlock) void ce_rows_prepare_kernel(const float *__restrict__ x, int64_t K, const Labels labels, int blocks_n, int64_t groups,
                                                                 int64_t blocks_k, u32x4 *__restrict__ by_n, u32x4 *__restrict__ by_k, float *saved)
{
    if (saved && blockIdx.x == 0 && threadIdx.x == 0)
        reinterpret_cast<int *>(saved)[kTicket] = 0;
    const int lane = threadIdx.x & 63;
    const int64_t unit = (int64_t)blockIdx.x * (kBlock / 64) + (threadIdx.x >> 6);
    float v[8];
    if (by_n && unit < groups * blocks_n)
    {
        const int64_t g = unit / blocks_n, n = (unit - g * blocks_n) * 32 + (lane & 31), k = g * 16 + (lane >> 5) * 8;
        const bool counts = labels(n) >= 0;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            v[e] = counts && k + e < K ? x[n * K + k + e] : 0.f;
        store3(by_n + unit * kFragment, v, lane);
    }
    if (by_k && unit < blocks_k * blocks_n * 2)
    {
        const int64_t kb = unit / (blocks_n * 2), k = kb * 32 + (lane & 31), n0 = (unit - kb * blocks_n * 2) * 16 + (lane >> 5) * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            v[e] = k < K && labels(n0 + e) >= 0 ? x[(n0 + e) * K + k] : 0.f;
        store3(by_k + unit * kFragment, v, lane);
    }
}

struct Stream
{
    const float *w;
    int64_t ld, outs, contraction;
    const u32x4 *q;       // the small operand, [groups][blocks_n]
    int blocks_n;         // its blocks of 32 rows; a workgroup takes NB of them
    int64_t groups;       // steps of 16 contraction values
    int64_t wave_groups;  // steps of one wave
};

// OUT_ROWS: w is [out][contraction], else [contraction][out]. A workgroup has 32 * VB outputs and 32 * NB rows; output of row r of
// block m: 32m + r (OUT_ROWS) or VB * r + m. The epilogue is called by all waves; waves m < VB hold block m, element 4q + e of
// s[nb] being row 8q + 4 * (lane / 32) + e, column nb * 32 + lane % 32.
template <int VB, int NB, bool OUT_ROWS, class Epilogue>
__global__ __launch_bounds__(64 * kWaves, 2) void ce_stream_kernel(const Stream a, const Epilogue epilogue)
{
    typedef float wide __attribute__((ext_vector_type(VB), aligned(4)));   // rows of w need not start on 16 bytes
    typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
    constexpr int kTile = 32 * VB, kReduce = kWaves * VB * 4096, kRows = kTile * (32 * NB + 1) * 4;
    __shared__ __attribute__((aligned(16))) char lds[kReduce > kRows ? kReduce : kRows];
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31;
    // workgroups with the same part of w are neighbours
    const unsigned per_tile = (unsigned)(a.blocks_n / NB);
    const unsigned tile     = blockIdx.x / per_tile;
    const int nb0           = (int)(blockIdx.x - tile * per_tile) * NB;
    const int64_t o0        = (int64_t)tile * kTile;
    f32x16 acc[VB][NB];
#pragma unroll
    for (int m = 0; m < VB; ++m)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                acc[m][nb][e] = 0.f;
    // Along rows of w the waves take steps in turn: together they read 512 consecutive bytes of a row (one row over
    // [32000, 1024]: 40 us; with an eighth of the row each, 64 bytes at a time, 54). Down columns each takes rows of its own.
    // (Workgroups that start at different places of their rows were slower, [100000, 2048]: 251 -> 283 us.)
    constexpr int kTurn  = OUT_ROWS ? kWaves : 1;
    const int64_t base   = (int64_t)blockIdx.y * kWaves * a.wave_groups;
    const int64_t first  = base + (OUT_ROWS ? wave : wave * a.wave_groups);
    const int64_t last   = min(OUT_ROWS ? base + kWaves * a.wave_groups : first + a.wave_groups, a.groups);
    const int64_t whole = a.outs >= VB || OUT_ROWS ? min(last, a.contraction / 16) : first;
    // In the last tile a lane past the outputs reads what lies in reach instead (its outputs are nobody's); of outputs that
    // straddle the end it reads the last VB and moves them to their places.
    const int64_t o_lane = o0 + col * VB, shift = OUT_ROWS ? 0 : o_lane + VB - a.outs;
    const bool straddles = !OUT_ROWS && o0 + kTile > a.outs;
    const float *w[VB];
#pragma unroll
    for (int m = 0; m < VB; ++m)
        w[m] = OUT_ROWS ? a.w + min(o0 + 32 * m + col, a.outs - 1) * a.ld + half * 8 : a.w + (int64_t)(half * 8) * a.ld + (shift > 0 ? a.outs - VB : o_lane);
    const u32x4 *q = a.q + (int64_t)nb0 * kFragment + lane;
    struct Step
    {
        float v[VB][8];  // block m's eight contraction values
    };
    const auto load = [&](int64_t g, Step &s) {
        const int64_t at = min(g, whole - 1);  // past the wave's last whole step: that one again, multiplied by nobody
        if constexpr (OUT_ROWS)
        {
#pragma unroll
            for (int m = 0; m < VB; ++m)
            {
                const f32x4 lo = *reinterpret_cast<const f32x4u *>(w[m] + at * 16), hi = *reinterpret_cast<const f32x4u *>(w[m] + at * 16 + 4);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    s.v[m][e] = lo[e], s.v[m][4 + e] = hi[e];
            }
        }
        else
        {
#pragma unroll
            for (int e = 0; e < 8; ++e)
            {
                const wide r = *reinterpret_cast<const wide *>(w[0] + (at * 16 + e) * a.ld);
#pragma unroll
                for (int m = 0; m < VB; ++m)
                    s.v[m][e] = r[m];
            }
        }
    };
    // the contraction's last values, single loads with zeros past its end (and outputs fewer than VB)
    const auto load_guarded = [&](int64_t g, Step &s) {
#pragma unroll
        for (int m = 0; m < VB; ++m)
#pragma unroll
            for (int e = 0; e < 8; ++e)
            {
                const int64_t o = OUT_ROWS ? o0 + 32 * m + col : o0 + col * VB + m, c = g * 16 + half * 8 + e;
                s.v[m][e] = o < a.outs && c < a.contraction ? a.w[OUT_ROWS ? o * a.ld + c : c * a.ld + o] : 0.f;
            }
    };
    const auto load_q = [&](int64_t g, u32x4 (*b)[3]) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int p = 0; p < 3; ++p)
                b[nb][p] = q[(g * a.blocks_n + nb) * kFragment + p * 64];
    };
    const auto step = [&](Step &s, const u32x4 (*b)[3], bool move) {
        if (move)
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int i = 1; i < VB; ++i)
                    if (shift == i)
                    {
#pragma unroll
                        for (int m = 0; m < VB; ++m)
                            s.v[m][e] = m + i < VB ? s.v[m + i < VB ? m + i : m][e] : 0.f;
                    }
#pragma unroll
        for (int m = 0; m < VB; ++m)
        {
            u32x4 part[3];
            split3(s.v[m], part);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
                multiply(acc[m][nb], part, b[nb]);
        }
    };
    if (first < whole)
    {
        Step s0, s1;
        u32x4 b[NB][3];
        load(first, s0);
        for (int64_t g = first; g < whole; g += 2 * kTurn)
        {
            load_q(g, b);
            load(g + kTurn, s1);
            step(s0, b, straddles);
            if (g + kTurn < whole)
            {
                load_q(g + kTurn, b);
                load(g + 2 * kTurn, s0);
                step(s1, b, straddles);
            }
        }
    }
    for (int64_t g = first < whole ? first + (whole - first + kTurn - 1) / kTurn * kTurn : first; g < last; g += kTurn)
    {
        Step s;
        u32x4 b[NB][3];
        load_q(g, b);
        load_guarded(g, s);
        step(s, b, false);
    }
    // the waves' sums, one block of columns at a time; wave m < VB adds up block m in the waves' order
    f32x4 *sums = reinterpret_cast<f32x4 *>(lds);
    f32x16 sum[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
    {
        if (nb)
            __syncthreads();
#pragma unroll
        for (int m = 0; m < VB; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                sums[(wave * VB + m) * 256 + i * 64 + lane] = f32x4{acc[m][nb][4 * i], acc[m][nb][4 * i + 1], acc[m][nb][4 * i + 2], acc[m][nb][4 * i + 3]};
        __syncthreads();
        if (wave < VB)
        {
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
                f32x4 v = sums[wave * 256 + i * 64 + lane];
#pragma unroll
                for (int u = 1; u < kWaves; ++u)
                    v += sums[(u * VB + wave) * 256 + i * 64 + lane];
                sum[nb][4 * i] = v[0], sum[nb][4 * i + 1] = v[1], sum[nb][4 * i + 2] = v[2], sum[nb][4 * i + 3] = v[3];
            }
        }
    }
    __syncthreads();  // the epilogue writes LDS
    epilogue.template run<VB, NB, OUT_ROWS>(tile, nb0, a.blocks_n, wave, lane, sum, reinterpret_cast<float *>(lds));
}

// place in the tile of element e of a lane's block m
template <int VB, bool OUT_ROWS>
__device__ inline int place_of(int m, int lane, int e)
{
    const int r = 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
    return OUT_ROWS ? 32 * m + r : VB * r + m;
}

// Where a workgroup of waves m keeps its sums between the passes: [tile][workgroup of rows][block of rows][block of outputs], each
// as a wave holds it. (The address need not be a multiple of 16.)
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
template <int VB, int NB, class F>
__device__ inline F *kept_at(F *kept, int64_t tile, int nb0, int blocks_n, int nb, int m, int lane)
{
    return kept + ((tile * (blocks_n / NB) + nb0 / NB) * NB + nb) * (VB * 1024) + m * 1024 + lane * 4;
}

struct RowsStatsEpilogue
{
    const float *b;
    Labels labels;
    int64_t v0, V;  // the launch's first entry, and how many it has
    float *part_m, *part_s, *target;
    float *kept;  // null, or where x.w stays for the backward pass (rows past the batch are left out)
    template <int VB, int NB, bool OUT_ROWS>
    __device__ void run(int64_t tile, int nb0, int blocks_n, int m, int lane, f32x16 *z, float *lds) const
    {
        float *lm = lds, *ls = lds + VB * NB * 32;
        if (m < VB)
        {
            float bias[16];
#pragma unroll
            for (int e = 0; e < 16; ++e)
            {
                const int64_t v = tile * (32 * VB) + place_of<VB, OUT_ROWS>(m, lane, e);
                bias[e] = v < V ? (b ? b[v] : 0.f) : -INFINITY;
            }
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
            {
                const int64_t n = (nb0 + nb) * 32 + (lane & 31), label = labels(n) - v0 - tile * (32 * VB);
                float top = -INFINITY;
                if (kept && n < labels.N)
                {
                    float *at = kept_at<VB, NB>(kept, tile, nb0, blocks_n, nb, m, lane);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        *reinterpret_cast<f32x4u *>(at + i * 256) = f32x4{z[nb][4 * i], z[nb][4 * i + 1], z[nb][4 * i + 2], z[nb][4 * i + 3]};
                }
#pragma unroll
                for (int e = 0; e < 16; ++e)
                {
                    // (past the vocabulary anything may have been read: selected away, not added to)
                    z[nb][e] = bias[e] == -INFINITY ? -INFINITY : z[nb][e] + bias[e];
                    if (place_of<VB, OUT_ROWS>(m, lane, e) == label)
                        target[n] = z[nb][e];
                    top = fmaxf(top, z[nb][e]);
                }
                float s = 0.f;
                const float sub = finite_top(top);
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    s += exp_under(z[nb][e], sub);
                const float top_o = __shfl_xor(top, 32, 64), s_o = __shfl_xor(s, 32, 64);
                merge(top, s, top_o, s_o);
                if (lane < 32)
                    lm[m * NB * 32 + nb * 32 + lane] = top, ls[m * NB * 32 + nb * 32 + lane] = s;
            }
        }
        __syncthreads();
        if (threadIdx.x < NB * 32)
        {
            const int n = threadIdx.x;
            float top = lm[n], s = ls[n];
#pragma unroll
            for (int i = 1; i < VB; ++i)
                merge(top, s, lm[i * NB * 32 + n], ls[i * NB * 32 + n]);
            const int64_t at = tile * (blocks_n * 32) + nb0 * 32 + n;
            part_m[at] = top, part_s[at] = s;
        }
    }
};

// d / counted rows (the mean first: the rows' sum of d x may be out of range) of a piece of the vocabulary, split: by_n as the small
// operand of gx, [V / 16][blocks of 32 rows]; by_v as an operand of gw, rows of the vocabulary, [V / 32][rows / 16] (null: not
// wanted); and the sums over this workgroup's rows for gb
struct RowsGradEpilogue
{
    const float *b, *saved, *row;
    Labels labels;
    int64_t v0, V;  // the piece's first entry, and how many it has
    u32x4 *by_n, *by_v;
    float *sums;  // [V padded to tiles][workgroups of rows]
    template <int VB, int NB, bool OUT_ROWS>
    __device__ void run(int64_t tile, int nb0, int blocks_n, int m, int lane, f32x16 *z, float *lds) const
    {
        constexpr int kTile = 32 * VB, kPitch = 32 * NB + 1;
        if (m < VB)
        {
            const float share = 1.f / fmaxf(saved[kCounted], 1.f);
            float bias[16];
#pragma unroll
            for (int e = 0; e < 16; ++e)
            {
                const int64_t v = tile * kTile + place_of<VB, OUT_ROWS>(m, lane, e);
                bias[e] = v < V && b ? b[v] : 0.f;
            }
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
            {
                const int64_t n = (nb0 + nb) * 32 + (lane & 31), label = labels(n);
                const bool counts = label >= 0;
                const float top = counts ? row[2 * n] : 0.f, inv = counts ? 1.f / row[2 * n + 1] : 0.f;
#pragma unroll
                for (int e = 0; e < 16; ++e)
                {
                    const int at    = place_of<VB, OUT_ROWS>(m, lane, e);
                    const int64_t v = tile * kTile + at;
                    float d = 0.f;
                    if (counts && v < V)
                    {
                        d = exp_under(z[nb][e] + bias[e], top) * inv;
                        if (v == label - v0)
                            d -= 1.f;
                        d *= share;
                    }
                    lds[at * kPitch + nb * 32 + (lane & 31)] = d;
                }
            }
        }
        __syncthreads();
        float v[8];
        if (by_n)
            for (int f = m; f < 2 * VB * NB; f += kWaves)
            {
                const int g = f / NB, nb = f % NB;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    v[e] = lds[(g * 16 + (lane >> 5) * 8 + e) * kPitch + nb * 32 + (lane & 31)];
                store3(by_n + ((tile * (2 * VB) + g) * blocks_n + nb0 + nb) * kFragment, v, lane);
            }
        if (by_v)
            for (int f = m; f < 2 * VB * NB; f += kWaves)
            {
                const int vb = f / (2 * NB), kb = f % (2 * NB);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    v[e] = lds[(vb * 32 + (lane & 31)) * kPitch + kb * 16 + (lane >> 5) * 8 + e];
                store3(by_v + ((tile * VB + vb) * blocks_n * 2 + nb0 * 2 + kb) * kFragment, v, lane);
            }
        if (sums && threadIdx.x < kTile)
        {
            // sixteen sums and a tree over them: a long chain would round every time
            float part[16];
#pragma unroll
            for (int i = 0; i < 16; ++i)
                part[i] = lds[threadIdx.x * kPitch + i];
            for (int n = 16; n < 32 * NB; n += 16)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    part[i] += lds[threadIdx.x * kPitch + n + i];
#pragma unroll
            for (int o = 8; o > 0; o >>= 1)
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i < o)
                        part[i] += part[i + o];
            const float s = part[0];
            sums[(tile * kTile + threadIdx.x) * (blocks_n / NB) + nb0 / NB] = s;
        }
    }
};

// the pass over w for the logits, where the forward pass has kept them
template <int VB, int NB, bool OUT_ROWS, class Epilogue>
__global__ __launch_bounds__(64 * kWaves) void ce_kept_kernel(const float *__restrict__ kept, int blocks_n, const Epilogue epilogue)
{
    __shared__ float lds[32 * VB * (32 * NB + 1)];
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63;
    const unsigned per_tile = (unsigned)(blocks_n / NB), tile = blockIdx.x / per_tile;
    const int nb0 = (int)(blockIdx.x - tile * per_tile) * NB;
    f32x16 sum[NB];
    if (wave < VB)
    {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
                const f32x4 v  = *reinterpret_cast<const f32x4u *>(kept_at<VB, NB>(kept, tile, nb0, blocks_n, nb, wave, lane) + i * 256);
                sum[nb][4 * i] = v[0], sum[nb][4 * i + 1] = v[1], sum[nb][4 * i + 2] = v[2], sum[nb][4 * i + 3] = v[3];
            }
    }
    epilogue.template run<VB, NB, OUT_ROWS>(tile, nb0, blocks_n, wave, lane, sum, lds);
}

// parts[run][feature][rows], (+)= over the pieces of the vocabulary
struct RowsPartEpilogue
{
    float *parts;
    int64_t outs;
    int add;
    template <int VB, int NB, bool OUT_ROWS>
    __device__ void run(int64_t tile, int nb0, int blocks_n, int m, int lane, f32x16 *z, float *) const
    {
        if (m >= VB)
            return;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int e = 0; e < 16; ++e)
            {
                const int64_t o = tile * (32 * VB) + place_of<VB, OUT_ROWS>(m, lane, e);
                if (o < outs)
                {
                    float *at = parts + ((int64_t)blockIdx.y * outs + o) * (blocks_n * 32) + (nb0 + nb) * 32 + (lane & 31);
                    *at       = add ? *at + z[nb][e] : z[nb][e];
                }
            }
    }
};

__global__ __launch_bounds__(kBlock) void ce_rows_gb_kernel(const float *__restrict__ sums, int groups, int64_t V, const float *gy, float *__restrict__ gb)
{
    const int64_t v = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (v >= V)
        return;
    float s = sums[v * groups];
    for (int i = 1; i < groups; ++i)
        s += sums[v * groups + i];
    gb[v] = gy ? s * *gy : s;
}

// gx[n][k] = gy * the runs' sums, in order; a workgroup takes 32 features and 32 rows
__global__ __launch_bounds__(kBlock) void ce_rows_gx_kernel(const float *__restrict__ parts, int runs, int64_t N, int64_t K, int rows, const float *gy,
                                                            float *__restrict__ gx)
{
    __shared__ float tile[32][33];
    const float g = gy ? *gy : 1.f;
    const int64_t k0 = (int64_t)blockIdx.x * 32, n0 = (int64_t)blockIdx.y * 32;
    for (int i = threadIdx.x; i < 32 * 32; i += kBlock)
    {
        const int k = i / 32, n = i % 32;
        float s = 0.f;
        if (k0 + k < K)
#pragma unroll 8
            for (int r = 0; r < runs; ++r)
                s += parts[((int64_t)r * K + k0 + k) * rows + n0 + n];
        tile[k][n] = s * g;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * 32; i += kBlock)
    {
        const int n = i / 32, k = i % 32;
        if (n0 + n < N && k0 + k < K)
            gx[(n0 + n) * K + k0 + k] = tile[k][n];
    }
}

// gw = gy * d^T.x over the rows: out[r][c] from operands split by r and by c, [blocks of 32][rows / 16]. A wave makes 32 rows of 128
// columns; the four waves of a workgroup share the columns' operand, and walk down `steps` blocks of 128 rows.
__global__ __launch_bounds__(kBlock, 2) void ce_rows_outer_kernel(const u32x4 *__restrict__ by_r, const u32x4 *__restrict__ by_c, int kbs, int64_t rows, int64_t cols, int64_t ld,
                                                                  unsigned tiles_c, int steps, const float *gy, float *__restrict__ out)
{
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const float g = gy ? *gy : 1.f;
    const unsigned group = blockIdx.x / tiles_c;
    const int64_t c0 = (int64_t)(blockIdx.x - group * tiles_c) * 128;
    for (int step = 0; step < steps; ++step)
    {
        const int64_t r0 = (((int64_t)group * steps + step) * 4 + wave) * 32;
        if (r0 >= rows)
            return;
        const u32x4 *r = by_r + r0 / 32 * kbs * kFragment + lane, *c = by_c + c0 / 32 * kbs * kFragment + lane;
        f32x16 acc[4];
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                acc[m][e] = 0.f;
#pragma unroll 2
        for (int kb = 0; kb < kbs; ++kb)
        {
            u32x4 a[3], b[4][3];
#pragma unroll
            for (int p = 0; p < 3; ++p)
                a[p] = r[kb * kFragment + p * 64];
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int p = 0; p < 3; ++p)
                    b[m][p] = c[(m * kbs + kb) * kFragment + p * 64];
#pragma unroll
            for (int m = 0; m < 4; ++m)
                multiply(acc[m], a, b[m]);
        }
#pragma unroll
        for (int m = 0; m < 4; ++m)
        {
            const int64_t col = c0 + m * 32 + (lane & 31);
            if (col >= cols)
                continue;
#pragma unroll
            for (int e = 0; e < 16; ++e)
            {
                const int64_t row = r0 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
                if (row < rows)
                    out[row * ld + col] = acc[m][e] * g;
            }
        }
    }
}

// blocks of 32 rows that a call's rows take, and how many a workgroup of a stream has: 1, 2 or 4
int blocks_of(int64_t N)
{
    return N <= 32 ? 1 : N <= 64 ? 2 : N <= 128 ? 4 : 8;
}
int taken_of(int blocks_n)
{
    return std::min(blocks_n, 4);
}
// outputs of a stream's workgroup: accumulators of 128 x 64 or 64 x 128
int64_t tile_of(int blocks_n)
{
    return taken_of(blocks_n) == 4 ? 64 : 128;
}

// fragments of an operand with `rows` rows: whole tiles of 128, so that what a stream or a tile of gw reaches is there
size_t fragments_bytes(int64_t rows, int64_t blocks_n)
{
    return (size_t)odl::ceil_div(rows, 128) * 8 * (size_t)blocks_n * kFragment * 16;
}

// Entries of the vocabulary whose d, as both operands of its products, stays within 512 MB: whole tiles, in equal pieces.
int64_t piece_of(int64_t V, int blocks_n)
{
    const int64_t most = ((int64_t)1 << 29) / (2 * 6 * 32 * blocks_n) / 128 * 128, pieces = odl::ceil_div(V, most);
    return pieces == 1 ? V : odl::ceil_div(odl::ceil_div(V, pieces), 128) * 128;
}

int runs_for_gx(int64_t K, int64_t V, int blocks_n)
{
    const int64_t groups = odl::ceil_div(K, tile_of(blocks_n)) * (blocks_n / taken_of(blocks_n));
    return (int)std::max<int64_t>(1, std::min<int64_t>(odl::device_cus() / groups, odl::ceil_div(V, 256)));
}

struct FewSpace
{
    u32x4 *x_by_n, *x_by_k, *d_by_n, *d_by_v;
    float *part_m, *part_s, *target, *parts, *sums;
    void *join_scratch;
    size_t bytes;
};

FewSpace forward_space(char *base, int64_t N, int64_t K, int64_t V)
{
    FewSpace s{};
    Carver c{base};
    const int blocks_n = blocks_of(N);
    const size_t rows = (size_t)blocks_n * 32, tiles = (size_t)odl::ceil_div(V, tile_of(blocks_n));
    s.x_by_n       = c.take<u32x4>(fragments_bytes(K, blocks_n));
    s.part_m       = c.take<float>(tiles * rows * 4);
    s.part_s       = c.take<float>(tiles * rows * 4);
    s.target       = c.take<float>(rows * 4);
    s.join_scratch = c.take<void>(join_scratch_bytes(N));
    s.bytes        = c.used;
    return s;
}

FewSpace backward_space(char *base, int64_t N, int64_t K, int64_t V)
{
    FewSpace s{};
    Carver c{base};
    const int blocks_n  = blocks_of(N);
    const int64_t piece = piece_of(V, blocks_n);
    s.x_by_n = c.take<u32x4>(fragments_bytes(K, blocks_n));
    s.x_by_k = c.take<u32x4>(fragments_bytes(K, blocks_n));
    s.d_by_n = c.take<u32x4>(fragments_bytes(piece, blocks_n));
    s.d_by_v = c.take<u32x4>(fragments_bytes(piece, blocks_n));
    s.sums   = c.take<float>((size_t)odl::ceil_div(piece, 128) * 128 * 2 * 4);
    s.parts  = c.take<float>((size_t)runs_for_gx(K, piece, blocks_n) * (size_t)K * (size_t)blocks_n * 32 * 4);
    s.bytes  = c.used;
    return s;
}

// a launch's threads along x have to fit 32 bits
int check_blocks(int64_t blocks, int threads)
{
    ODL_REQUIRE(blocks <= ((int64_t)1 << 32) / threads - 1, "linear_softmax_ce: too many tiles");
    return ODL_OK;
}

template <class Epilogue>
int stream(const float *w, bool out_rows, int64_t ld, int64_t outs, int64_t contraction, const u32x4 *q, int blocks_n, int runs, const Epilogue &e, hipStream_t st)
{
    Stream a{w, ld, outs, contraction, q, blocks_n, odl::ceil_div(contraction, 16), 0};
    a.wave_groups = odl::ceil_div(a.groups, (int64_t)runs * kWaves);
    const int64_t blocks = odl::ceil_div(outs, tile_of(blocks_n)) * (blocks_n / taken_of(blocks_n));
    if (int rc = check_blocks(blocks, 64 * kWaves))
        return rc;
    const dim3 grid((unsigned)blocks, (unsigned)runs), block(64 * kWaves);
    switch (taken_of(blocks_n) * 2 + (out_rows ? 1 : 0))
    {
        case 2: ce_stream_kernel<4, 1, false, Epilogue><<<grid, block, 0, st>>>(a, e); break;
        case 3: ce_stream_kernel<4, 1, true, Epilogue><<<grid, block, 0, st>>>(a, e); break;
        case 4: ce_stream_kernel<4, 2, false, Epilogue><<<grid, block, 0, st>>>(a, e); break;
        case 5: ce_stream_kernel<4, 2, true, Epilogue><<<grid, block, 0, st>>>(a, e); break;
        case 8: ce_stream_kernel<2, 4, false, Epilogue><<<grid, block, 0, st>>>(a, e); break;
        default: ce_stream_kernel<2, 4, true, Epilogue><<<grid, block, 0, st>>>(a, e); break;
    }
    ODL_LAUNCH_CHECK();
    return ODL_OK;
}

template <class Epilogue>
int from_kept(const float *kept, bool out_rows, int64_t outs, int blocks_n, const Epilogue &e, hipStream_t st)
{
    const int64_t blocks = odl::ceil_div(outs, tile_of(blocks_n)) * (blocks_n / taken_of(blocks_n));
    if (int rc = check_blocks(blocks, 64 * kWaves))
        return rc;
    const dim3 grid((unsigned)blocks), block(64 * kWaves);
    switch (taken_of(blocks_n) * 2 + (out_rows ? 1 : 0))
    {
        case 2: ce_kept_kernel<4, 1, false, Epilogue><<<grid, block, 0, st>>>(kept, blocks_n, e); break;
        case 3: ce_kept_kernel<4, 1, true, Epilogue><<<grid, block, 0, st>>>(kept, blocks_n, e); break;
        case 4: ce_kept_kernel<4, 2, false, Epilogue><<<grid, block, 0, st>>>(kept, blocks_n, e); break;
        case 5: ce_kept_kernel<4, 2, true, Epilogue><<<grid, block, 0, st>>>(kept, blocks_n, e); break;
        case 8: ce_kept_kernel<2, 4, false, Epilogue><<<grid, block, 0, st>>>(kept, blocks_n, e); break;
        default: ce_kept_kernel<2, 4, true, Epilogue><<<grid, block, 0, st>>>(kept, blocks_n, e); break;
    }
    ODL_LAUNCH_CHECK();
    return ODL_OK;
}

// whole tiles of 128 features: a tile of gw reads them all
int prepare(const Problem &p, int blocks_n, u32x4 *by_n, u32x4 *by_k, float *saved, hipStream_t st)
{
    const int64_t groups = odl::ceil_div(p.K, 128) * 8, blocks_k = groups / 2;
    ce_rows_prepare_kernel<<<dim3((unsigned)odl::ceil_div(groups * blocks_n, kBlock / 64)), dim3(kBlock), 0, st>>>(p.x, p.K, p.labels, blocks_n, groups, blocks_k,
                                                                                                            by_n, by_k, saved);
    ODL_LAUNCH_CHECK();
    return ODL_OK;
}
}  // namespace

namespace odl
{
namespace linear_ce
{
size_t few_forward_bytes(int64_t N, int64_t K, int64_t V)
{
    return ::forward_space(nullptr, N, K, V).bytes;
}

size_t few_backward_bytes(int64_t N, int64_t K, int64_t V)
{
    return ::backward_space(nullptr, N, K, V).bytes;
}

// The logits stay where they are at most a quarter of the weights, which the backward pass would read again for them.
size_t few_kept_floats(int64_t N, int64_t K, int64_t V)
{
    const int64_t rows = blocks_of(N) * 32, tile = tile_of(blocks_of(N));
    return 4 * rows <= K ? (size_t)(ceil_div(V, tile) * tile * rows) : 0;
}

int few_forward(const Problem &p, float *saved, float *row_stats, char *workspace, hipStream_t st)
{
    const int blocks_n = blocks_of(p.N);
    const FewSpace s   = ::forward_space(workspace, p.N, p.K, p.V);
    if (int rc = prepare(p, blocks_n, s.x_by_n, nullptr, saved, st))
        return rc;
    float *kept = few_kept_floats(p.N, p.K, p.V) ? row_stats + 2 * p.N : nullptr;
    // as many entries in a launch as its threads along x can be counted in 32 bits: 2^27 or more
    const int64_t tile = tile_of(blocks_n), rows = blocks_n * 32, most = ((int64_t)1 << 22) / (blocks_n / taken_of(blocks_n)) * tile;
    for (int64_t v0 = 0; v0 < p.V; v0 += most)
    {
        const int64_t vn = std::min(most, p.V - v0), at = v0 * (p.w_out_in ? p.K : 1);
        const RowsStatsEpilogue e{p.b ? p.b + v0 : nullptr, p.labels, v0, vn, s.part_m + v0 / tile * rows, s.part_s + v0 / tile * rows, s.target,
                                  kept ? kept + v0 * rows : nullptr};
        if (int rc = stream(p.w + at, p.w_out_in != 0, p.w_out_in ? p.K : p.V, vn, p.K, s.x_by_n, blocks_n, 1, e, st))
            return rc;
    }
    return join(s.part_m, s.part_s, s.target, ceil_div(p.V, tile), rows, p.labels, row_stats, s.join_scratch, saved, st);
}

int few_backward(const Problem &p, const float *gy, const float *saved, const float *row_stats, float *gx, float *gw, float *gb, char *workspace,
                 hipStream_t st)
{
    const int blocks_n = blocks_of(p.N);
    const FewSpace s   = ::backward_space(workspace, p.N, p.K, p.V);
    const bool kept    = few_kept_floats(p.N, p.K, p.V) != 0;
    if (gw || !kept)
        if (int rc = prepare(p, blocks_n, kept ? nullptr : s.x_by_n, gw ? s.x_by_k : nullptr, nullptr, st))
            return rc;
    const int64_t ld = p.w_out_in ? p.K : p.V, piece = piece_of(p.V, blocks_n);
    const int runs = runs_for_gx(p.K, piece, blocks_n);
    for (int64_t v0 = 0; v0 < p.V; v0 += piece)
    {
        const int64_t vn = std::min(piece, p.V - v0), at = v0 * (p.w_out_in ? p.K : 1);
        const RowsGradEpilogue e{p.b ? p.b + v0 : nullptr, saved, row_stats, p.labels, v0, vn, gx ? s.d_by_n : nullptr, gw ? s.d_by_v : nullptr,
                                 gb ? s.sums : nullptr};
        if (int rc = kept ? from_kept(row_stats + 2 * p.N + v0 * (blocks_n * 32), p.w_out_in != 0, vn, blocks_n, e, st)
                          : stream(p.w + at, p.w_out_in != 0, ld, vn, p.K, s.x_by_n, blocks_n, 1, e, st))
            return rc;
        if (gb)
        {
            ce_rows_gb_kernel<<<dim3((unsigned)ceil_div(vn, kBlock)), dim3(kBlock), 0, st>>>(s.sums, blocks_n / taken_of(blocks_n), vn, gy, gb + v0);
            ODL_LAUNCH_CHECK();
        }
        if (gx)
            if (int rc = stream(p.w + at, p.w_out_in == 0, ld, p.K, vn, s.d_by_n, blocks_n, runs, RowsPartEpilogue{s.parts, p.K, v0 > 0}, st))
                return rc;
        if (gw)
        {
            const int64_t r = p.w_out_in ? vn : p.K, c = p.w_out_in ? p.K : vn;
            // enough workgroups for the chip, and as many rows each as that leaves: they share the columns' operand
            const int64_t tiles_c = ceil_div(c, 128), tiles_r = ceil_div(r, 128);
            const int steps = (int)std::max<int64_t>(1, std::min<int64_t>(16, tiles_c * tiles_r / (8 * (int64_t)device_cus())));
            const int64_t blocks = tiles_c * ceil_div(tiles_r, steps);
            if (int rc = check_blocks(blocks, kBlock))
                return rc;
            ce_rows_outer_kernel<<<dim3((unsigned)blocks), dim3(kBlock), 0, st>>>(p.w_out_in ? s.d_by_v : s.x_by_k, p.w_out_in ? s.x_by_k : s.d_by_v,
                                                                                 blocks_n * 2, r, c, ld, (unsigned)tiles_c, steps, gy, gw + at);
            ODL_LAUNCH_CHECK();
        }
    }
    if (gx)
    {
        ce_rows_gx_kernel<<<dim3((unsigned)ceil_div(p.K, 32), (unsigned)blocks_n), dim3(kBlock), 0, st>>>(s.parts, runs, p.N, p.K, blocks_n * 32, gy, gx);
        ODL_LAUNCH_CHECK();
    }
    return ODL_OK;
}
}  // namespace linear_ce
}  // namespace odl
