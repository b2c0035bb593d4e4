// A linear layer and its softmax cross-entropy as one operator, forward and backward, for vocabularies whose logits are not
// to be stored: z[n][v] = x[n].w[v] + b[v] exists only as accumulators.
//
//   forward   per 256 (128, 64) vocabulary entries and token: m = max z and s = sum e^(z - m), formed in the product's epilogue;
//             one launch joins them per token: loss_n = m + ln(s) - z[n][t_n]
//   backward  the vocabulary in pieces: the logits of a piece again, d = e^(z - m) / s - [v = t_n] from the accumulators,
//             written as the operands of the two products that follow (rows of tokens for gx += d.w, rows of vocabulary for
//             gw = d^T.x); the sums over tokens for gb come out of the same epilogue.
//
// What bounds it: matrix products, 2NKV operations forward and 6NKV backward (the logits a second time: 4NKV with logits
// kept), each as three float16 products (split_gemm.h). Exponentials: one per logit and direction. Measured, 16384 tokens x 1024
// over 32000 entries: loss 2.63 to 2.74 ms, 392 to 408 TFLOP/s of all, 0.17 ms of it to find scales, lay out operands and join;
// 4096 tokens, both directions: 2.97 to 3.06 ms, of it 0.17 to lay out and 0.05 for sums and joins. The rest are products at
// the rate that the chip's power allows.
//
// In the products the vocabulary is the row side: a lane's accumulators then belong to one token, and the maximum and the
// sum over the vocabulary are sums over a lane's own registers, one exchange between the wave's halves and one through LDS.
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "linear_ce.h"
#include "split_gemm.h"

namespace
{
using namespace odl::split;
using namespace odl::linear_ce;

__device__ inline float block_max(float v, float *scratch)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        v = fmaxf(v, __shfl_xor(v, o, 64));
    if ((threadIdx.x & 63) == 0)
        scratch[threadIdx.x >> 6] = v;
    __syncthreads();
    v = fmaxf(fmaxf(scratch[0], scratch[1]), fmaxf(scratch[2], scratch[3]));
    __syncthreads();
    return v;
}

// The largest finite magnitudes of x's counted rows and of w, one per workgroup: the first `blocks_x` workgroups share x, the
// others w. Rows that do not count may hold anything. Also clears the ticket of the joining launch.
__global__ __launch_bounds__(kBlock) void ce_magnitudes_kernel(const float *__restrict__ x, int64_t N, int64_t K, const Labels labels,
                                                               const float *__restrict__ w, int64_t n_w, int blocks_x, float *out, float *saved)
{
    __shared__ float scratch[4];
    float m = 0.f;
    const auto take = [&](float v) {
        const float a = fabsf(v);
        m = a <= FLT_MAX ? fmaxf(m, a) : m;
    };
    if ((int)blockIdx.x < blocks_x)
    {
        const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
        for (int64_t n = (int64_t)blockIdx.x * 4 + wave; n < N; n += (int64_t)blocks_x * 4)
            if (labels(n) >= 0)
                for (int64_t k = lane; k < K; k += 64)
                    take(x[n * K + k]);
    }
    else
    {
        const int64_t step = (int64_t)(gridDim.x - blocks_x) * kBlock, at = (int64_t)(blockIdx.x - blocks_x) * kBlock + threadIdx.x;
        if ((reinterpret_cast<uintptr_t>(w) & 15) == 0)
        {
            for (int64_t i = at; i < n_w / 4; i += step)
            {
                const f32x4 v = reinterpret_cast<const f32x4 *>(w)[i];
                take(v[0]), take(v[1]), take(v[2]), take(v[3]);
            }
            for (int64_t i = n_w / 4 * 4 + at; i < n_w; i += step)
                take(w[i]);
        }
        else
            for (int64_t i = at; i < n_w; i += step)
                take(w[i]);
    }
    m = block_max(m, scratch);
    if (threadIdx.x == 0)
        out[blockIdx.x] = m;
    if (blockIdx.x == 0 && threadIdx.x == 0)
        reinterpret_cast<int *>(saved)[kTicket] = 0;
}

// the power of two that brings magnitude m to [2^14, 2^15): float16 holds it, and what is 2^17 times smaller keeps its bits (a
// largest magnitude under 2^-106 is brought less far, its operand's elements are kept to 2^-145)
__device__ inline float scale_for(float m)
{
    if (!(m > 0.f))
        return 1.f;
    int e;
    frexpf(m, &e);  // m = f * 2^e, f in [0.5, 1)
    e = 15 - e;
    return ldexpf(1.f, e > 120 ? 120 : e < -120 ? -120 : e);
}

__device__ inline float scale_from(const float *mags, int n, float *scratch)
{
    float m = 0.f;
    for (int i = threadIdx.x; i < n; i += kBlock)
        m = fmaxf(m, mags[i]);
    return scale_for(block_max(m, scratch));
}

// One launch lays out everything a pass multiplies: workgroups [0, x_tiles) x, then w's piece, then the piece's bias row
// (padded with -inf: entries past the vocabulary get probability 0 without a test).
struct PrepArgs
{
    const float *x, *w, *b;
    int64_t N, K, V;
    int w_out_in;
    int64_t v0, vn;              // the piece of the vocabulary
    Panel xr, xt, wr, wt;        // x: rows of tokens, rows of K; w: rows of vocabulary, rows of K (null base: not wanted)
    int x_tiles_r, x_tiles_c;    // 64 x 64 tiles of x's padded extents (0: x is laid out already)
    int w_tiles_r, w_tiles_c;    // of the piece's, in the order w lies
    int bias_blocks;             // 256 padded entries of the piece each
    float *bias;
    Labels labels;
    const float *mags;           // null: the scales are in saved[] already
    int mags_x, mags_w;
    float *saved;
};

struct XSource
{
    const float *x;
    int64_t K;
    Labels labels;
    __device__ float operator()(int64_t n, int64_t k) const
    {
        if (labels(n) < 0)
            return 0.f;  // a row that does not count may hold NaN: nothing of it enters a sum
        return x[n * K + k];
    }
};
struct WSource
{
    const float *w;
    int64_t ld, col0;
    __device__ float operator()(int64_t r, int64_t c) const { return w[r * ld + col0 + c]; }
};

__global__ __launch_bounds__(kBlock) void ce_prepare_kernel(const PrepArgs a)
{
    __shared__ float tile[64][65];
    __shared__ float scratch[4];
    int bid = (int)blockIdx.x;
    const int nx = a.x_tiles_r * a.x_tiles_c, nw = a.w_tiles_r * a.w_tiles_c;
    if (bid < nx)
    {
        const auto factor = [&] {
            const float s = a.mags ? scale_from(a.mags, a.mags_x, scratch) : a.saved[kScaleX];
            if (a.mags && blockIdx.x == 0 && threadIdx.x == 0)
                a.saved[kScaleX] = s;
            return s;
        };
        split_tile(XSource{a.x, a.K, a.labels}, factor, a.N, a.K, (int64_t)(bid / a.x_tiles_c) * 64, (int64_t)(bid % a.x_tiles_c) * 64, a.xr,
                   a.xt, tile);
        return;
    }
    bid -= nx;
    if (bid < nw)
    {
        const auto factor = [&] {
            const float s = a.mags ? scale_from(a.mags + a.mags_x, a.mags_w, scratch) : a.saved[kScaleW];
            if (a.mags && bid == 0 && threadIdx.x == 0)
                a.saved[kScaleW] = s;
            return s;
        };
        const int64_t r0 = (int64_t)(bid / a.w_tiles_c) * 64, c0 = (int64_t)(bid % a.w_tiles_c) * 64;
        if (a.w_out_in)
            split_tile(WSource{a.w + a.v0 * a.K, a.K, 0}, factor, a.vn, a.K, r0, c0, a.wr, a.wt, tile);
        else
            split_tile(WSource{a.w, a.V, a.v0}, factor, a.K, a.vn, r0, c0, a.wt, a.wr, tile);
        return;
    }
    bid -= nw;
    const int64_t v = (int64_t)bid * kBlock + threadIdx.x;
    const int64_t v_pad = (int64_t)(a.w_out_in ? a.w_tiles_r : a.w_tiles_c) * 64;
    if (v < v_pad)
        a.bias[v] = v < a.vn ? (a.b ? a.b[a.v0 + v] : 0.f) : -INFINITY;
}

// what takes the operands' scales out of a logit, the smaller factor first: the other one alone may lift it out of range
struct Unscale
{
    float first, second;
    __device__ explicit Unscale(const float *saved)
    {
        const float x = 1.f / saved[kScaleX], w = 1.f / saved[kScaleW];
        first = fminf(x, w), second = fmaxf(x, w);
    }
};

// a lane's logits of one accumulator block, rows as to_columns leaves them
__device__ inline void logits_of(f32x16 &c, const Unscale &by, const float *bias, int lane)
{
    to_columns(c);
    const float *b = bias + (lane >> 5) * 8;
#pragma unroll
    for (int h = 0; h < 2; ++h)
    {
        const f32x4 b0 = *reinterpret_cast<const f32x4 *>(b + 16 * h), b1 = *reinterpret_cast<const f32x4 *>(b + 16 * h + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e)
        {
            c[8 * h + e]     = c[8 * h + e] * by.first * by.second + b0[e];
            c[8 * h + 4 + e] = c[8 * h + 4 + e] * by.first * by.second + b1[e];
        }
    }
}

struct StatsEpilogue
{
    const float *bias;   // of the piece, padded
    const float *saved;
    Labels labels;
    int64_t v0;          // the piece's first entry
    int64_t n_pad;
    float *part_m, *part_s;  // [tile row][n_pad] of this piece
    float *target;       // [n_pad]: the label's logit
    template <class T, class Acc>
    __device__ void operator()(const T &t, Acc &acc) const
    {
        const Unscale by(saved);
        float *lm = reinterpret_cast<float *>(t.lds), *ls = lm + T::kWavesM * T::kCols;
#pragma unroll
        for (int ni = 0; ni < T::NI; ++ni)
        {
            const int64_t n = t.col_block(ni) * 32 + (t.lane & 31);
            const int64_t label = labels(n) - v0;
            float m = -INFINITY, s = 0.f;
#pragma unroll
            for (int mi = 0; mi < T::MI; ++mi)
            {
                const int64_t v = t.row_block(mi) * 32;
                f32x16 &c = acc[mi][ni];
                logits_of(c, by, bias + v, t.lane);
                if (label >= v && label < v + 32)
                {
                    const int at = (int)(label - v) - 8 * (t.lane >> 5);
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (at == (e & 7) + 16 * (e >> 3))
                            target[n] = c[e];
                }
                float top = c[0];
#pragma unroll
                for (int e = 1; e < 16; ++e)
                    top = fmaxf(top, c[e]);
                m = fmaxf(m, top);
            }
            const float sub = finite_top(m);
#pragma unroll
            for (int mi = 0; mi < T::MI; ++mi)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    s += exp_under(acc[mi][ni][e], sub);
            const float m_o = __shfl_xor(m, 32, 64), s_o = __shfl_xor(s, 32, 64);
            merge(m, s, m_o, s_o);
            if (t.lane < 32)
            {
                const int col = (t.wn * T::NI + ni) * 32 + t.lane;
                lm[t.wm * T::kCols + col] = m, ls[t.wm * T::kCols + col] = s;
            }
        }
        __syncthreads();
        for (int c = threadIdx.x; c < T::kCols; c += T::kWavesM * T::kWavesN * 64)
        {
            float m = lm[c], s = ls[c];
#pragma unroll
            for (int i = 1; i < T::kWavesM; ++i)
                merge(m, s, lm[i * T::kCols + c], ls[i * T::kCols + c]);
            const int64_t at = (int64_t)t.tm * n_pad + (int64_t)t.tn * T::kCols + c;
            part_m[at] = m, part_s[at] = s;
        }
    }
};

// Joins the partial maxima and sums of 16 tokens a workgroup, 16 threads a token; row[2n] = m, row[2n + 1] = s; the mean loss
// by the last workgroup to finish, which adds the workgroups' sums in their order.
constexpr int kJoinRows = 16;

__global__ __launch_bounds__(kBlock) void ce_join_kernel(const float *__restrict__ part_m, const float *__restrict__ part_s, const float *__restrict__ target,
                                                         int64_t tiles, int64_t n_pad, const Labels labels, float *__restrict__ row, double *block_loss,
                                                         int *block_count, float *saved)
{
    __shared__ float sm[4][kJoinRows];
    __shared__ double ss[4][kJoinRows];
    __shared__ int last;
    const int r = threadIdx.x % kJoinRows, g = threadIdx.x / kJoinRows;
    const int64_t n = (int64_t)blockIdx.x * kJoinRows + r;
    float m = -INFINITY;
    double s = 0.0;
#pragma unroll 8
    for (int64_t t = g; t < tiles; t += 16)
        merge(m, s, part_m[t * n_pad + n], (double)part_s[t * n_pad + n]);
    // a wave's four threads of a token, then the four waves
#pragma unroll
    for (int o = kJoinRows; o < 64; o *= 2)
    {
        const float m_o  = __shfl_xor(m, o, 64);
        const double s_o = __shfl_xor(s, o, 64);
        merge(m, s, m_o, s_o);
    }
    if ((threadIdx.x & 63) < kJoinRows)
        sm[threadIdx.x >> 6][r] = m, ss[threadIdx.x >> 6][r] = s;
    __syncthreads();
    if (threadIdx.x < 64)
    {
        double loss = 0.0;
        int count = 0, bad = 0;
        if (threadIdx.x < kJoinRows && n < labels.N)
        {
#pragma unroll
            for (int i = 1; i < 4; ++i)
                merge(m, s, sm[i][r], ss[i][r]);
            row[2 * n] = m, row[2 * n + 1] = (float)s;
            if (labels(n) >= 0)
                loss = (double)m - (double)target[n] + log(s), count = 1;
            else
                bad = label_of(labels.t, labels.is64, n) != labels.ignore;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1)
            loss += __shfl_xor(loss, o, 64), count += __shfl_xor(count, o, 64), bad |= __shfl_xor(bad, o, 64);
        if (threadIdx.x == 0)
        {
            block_loss[blockIdx.x] = loss, block_count[blockIdx.x] = bad ? ~count : count;
            __threadfence();
            last = atomicAdd(reinterpret_cast<int *>(saved) + kTicket, 1) == (int)gridDim.x - 1;
        }
    }
    __syncthreads();
    if (!last || threadIdx.x >= 64)
        return;
    __threadfence();
    double loss = 0.0;
    int count = 0, bad = 0;
    for (int b = threadIdx.x; b < (int)gridDim.x; b += 64)
    {
        const int c = block_count[b];
        loss += block_loss[b], count += c < 0 ? ~c : c, bad |= c < 0;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        loss += __shfl_xor(loss, o, 64), count += __shfl_xor(count, o, 64), bad |= __shfl_xor(bad, o, 64);
    if (threadIdx.x == 0)
    {
        saved[kLoss] = count ? (float)(loss / count) : 0.f;
        reinterpret_cast<int *>(saved)[kBadLabel] = bad;
        saved[kCounted] = (float)count;
    }
}

// d = softmax - one-hot of a tile, as operands of the two gradient products (times kDScale: float16's range)
struct GradEpilogue
{
    const float *bias, *saved, *row;
    Labels labels;
    int64_t v0;
    Panel dt, dr;   // rows of tokens, rows of vocabulary (null base: that product is not wanted)
    float *sums;    // [column waves of all tiles][v_pad]: d summed over a wave's tokens (null: no bias gradient)
    int64_t v_pad;
    template <class T, class Acc>
    __device__ void operator()(const T &t, Acc &acc) const
    {
        const Unscale by(saved);
        float *scratch = t.wave_scratch();
        float m[T::NI], inv_s[T::NI];
        int64_t label[T::NI];
        bool counts[T::NI];
#pragma unroll
        for (int ni = 0; ni < T::NI; ++ni)
        {
            const int64_t n = t.col_block(ni) * 32 + (t.lane & 31);
            label[ni]  = labels(n);
            counts[ni] = label[ni] >= 0;
            m[ni]      = counts[ni] ? row[2 * n] : 0.f;
            inv_s[ni]  = counts[ni] ? kDScale / row[2 * n + 1] : 0.f;
            label[ni] -= v0;
        }
#pragma unroll
        for (int mi = 0; mi < T::MI; ++mi)
        {
            const int64_t vb = t.row_block(mi);
            float sum = 0.f;
#pragma unroll
            for (int ni = 0; ni < T::NI; ++ni)
            {
                f32x16 &c = acc[mi][ni];
                logits_of(c, by, bias + vb * 32, t.lane);
                const int at = (int)(label[ni] - vb * 32) - 8 * (t.lane >> 5);
                const bool here = label[ni] >= vb * 32 && label[ni] < vb * 32 + 32;
#pragma unroll
                for (int e = 0; e < 16; ++e)
                {
                    float d = exp_under(c[e], m[ni]) * inv_s[ni];
                    if (here && at == (e & 7) + 16 * (e >> 3))
                        d -= kDScale;
                    c[e] = counts[ni] ? d : 0.f;  // by selection: the logits of a row that does not count may be anything
                }
                if (dt.base)
                {
                    float v[8];
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                    {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            v[e] = c[8 * h + e];
                        store_fragment(dt, t.col_block(ni), vb * 2 + h, t.lane, v);
                    }
                }
                if (dr.base || sums)
                {
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        scratch[(16 * (e >> 3) + 8 * (t.lane >> 5) + (e & 7)) * 33 + (t.lane & 31)] = c[e];
                    __builtin_amdgcn_wave_barrier();
                    float v[8];
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                    {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            v[e] = scratch[(t.lane & 31) * 33 + 16 * h + 8 * (t.lane >> 5) + e], sum += v[e];
                        if (dr.base)
                            store_fragment(dr, vb, t.col_block(ni) * 2 + h, t.lane, v);
                    }
                    __builtin_amdgcn_wave_barrier();
                }
            }
            if (sums)
            {
                sum += __shfl_xor(sum, 32, 64);
                if (t.lane < 32)
                    sums[((int64_t)t.tn * T::kWavesN + t.wn) * v_pad + vb * 32 + t.lane] = sum;
            }
        }
    }
};

// out[i][j] (+)= acc * gy / counted rows over the operands' scales. The mean is taken first: the rows' sum may be out of range.
struct OutEpilogue
{
    float *out;
    int64_t rows, cols, ld;
    int64_t split_stride;    // from one run of the contraction's results to the next one's
    const float *saved;
    int scale;               // kScaleX or kScaleW: whose scale the operand beside d carries
    const float *gy;
    int add;
    template <class T, class Acc>
    __device__ void operator()(const T &t, Acc &acc) const
    {
        const float g = (gy ? *gy : 1.f) / fmaxf(saved[kCounted], 1.f) / kDScale, inv = 1.f / saved[scale];
#pragma unroll
        for (int mi = 0; mi < T::MI; ++mi)
#pragma unroll
            for (int ni = 0; ni < T::NI; ++ni)
            {
                const int64_t col = t.col_block(ni) * 32 + (t.lane & 31);
                if (col >= cols)
                    continue;
#pragma unroll
                for (int e = 0; e < 16; ++e)
                {
                    const int64_t r = t.row_block(mi) * 32 + 8 * (e >> 2) + 4 * (t.lane >> 5) + (e & 3);
                    if (r < rows)
                    {
                        float *at = out + t.split * split_stride + r * ld + col;
                        const float v = acc[mi][ni][e] * g * inv;
                        *at = add ? *at + v : v;
                    }
                }
            }
    }
};

// What is added up after the products of a piece, in one launch. First gb[v]: the partial sums of the tiles' column waves in
// order, 64 entries a workgroup.
struct BiasGrad
{
    const float *sums;
    int parts;
    int64_t v_pad, vn;
    float *gb;
    const float *saved, *gy;
    __device__ void operator()(unsigned block) const
    {
        __shared__ float part[4][64];
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        const int64_t v = (int64_t)block * 64 + lane;
        float s = 0.f;
        for (int p = wave; p < parts; p += 4)
            s += sums[(int64_t)p * v_pad + v];
        part[wave][lane] = s;
        __syncthreads();
        if (wave == 0 && v < vn)
        {
            s = (part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]);
            gb[v] = s / kDScale * ((gy ? *gy : 1.f) / fmaxf(saved[kCounted], 1.f));
        }
    }
};

// Then, after the last piece, gx: the runs of the contraction in order, by the workgroups from bias_blocks on.
__global__ __launch_bounds__(kBlock) void ce_sums_kernel(const BiasGrad bias, unsigned bias_blocks, const float *__restrict__ parts, int count, int64_t n,
                                                         float *__restrict__ out)
{
    if (blockIdx.x < bias_blocks)
    {
        bias(blockIdx.x);
        return;
    }
    for (int64_t i = (int64_t)(blockIdx.x - bias_blocks) * kBlock + threadIdx.x; i < n; i += (int64_t)(gridDim.x - bias_blocks) * kBlock)
    {
        float s = parts[i];
        for (int p = 1; p < count; ++p)
            s += parts[(int64_t)p * n + i];
        out[i] = s;
    }
}

// How a call is cut: pieces of the vocabulary whose panels stay within a bound whatever V is.
struct Plan
{
    int64_t n_pad, k_pad, v_piece, pieces;
    Cut gx;  // of a whole piece; its runs of the contraction add up over the pieces, each in its own place
    int64_t vn(int64_t V, int64_t p) const { return std::min(v_piece, V - p * v_piece); }
};

Plan make_plan(int64_t N, int64_t K, int64_t V, bool backward)
{
    Plan p;
    p.n_pad = padded(N), p.k_pad = padded(K);
    // backward: d twice and w twice, 4 bytes an element; forward: w once
    const int64_t budget = (int64_t)1 << 26;
    int64_t most = backward ? std::min(budget / p.n_pad, budget / p.k_pad) : budget / p.k_pad;
    // a launch's threads have to fit 32 bits: one for 16 logits in the smallest tiles
    most = std::min(most, ((int64_t)1 << 35) / p.n_pad);
    most = std::max<int64_t>(most / 256 * 256, 1024);
    p.pieces  = odl::ceil_div(V, most);
    p.v_piece = p.pieces == 1 ? V : odl::ceil_div(odl::ceil_div(V, p.pieces), 256) * 256;
    p.pieces  = odl::ceil_div(V, p.v_piece);
    p.gx      = pick_cut(p.n_pad, p.k_pad, false, 1, contraction_blocks(p.v_piece), true, (double)N * (double)K * 4 / (double)p.pieces);
    return p;
}

int magnitude_blocks(int64_t elements)
{
    return (int)std::min<int64_t>(1024, std::max<int64_t>(1, odl::ceil_div(elements, 4096)));
}

struct ForwardSpace
{
    float *mags, *bias, *part_m, *part_s, *target;
    void *join_scratch;
    Panel xr, wr;
    size_t bytes;
};

ForwardSpace forward_space(char *base, const Plan &p, int64_t N, int64_t K, int64_t V)
{
    ForwardSpace s;
    Carver c{base};
    const int64_t v_pad = padded(p.v_piece);
    int64_t tiles = 0;  // of the vocabulary, over all pieces
    for (int64_t i = 0; i < p.pieces; ++i)
        tiles += padded(p.vn(V, i)) / pick_cut(padded(p.vn(V, i)), p.n_pad, false, 1, contraction_blocks(K)).bm;
    s.mags        = c.take<float>((size_t)(magnitude_blocks(N * K) + magnitude_blocks(K * V)) * 4);
    s.bias        = c.take<float>((size_t)v_pad * 4);
    s.part_m      = c.take<float>((size_t)(tiles * p.n_pad) * 4);
    s.part_s      = c.take<float>((size_t)(tiles * p.n_pad) * 4);
    s.target      = c.take<float>((size_t)p.n_pad * 4);
    s.join_scratch = c.take<void>(join_scratch_bytes(N));
    s.xr          = Panel{c.take<char>((size_t)panel_bytes(p.n_pad, p.k_pad)), p.k_pad / 16};
    s.wr          = Panel{c.take<char>((size_t)panel_bytes(v_pad, p.k_pad)), p.k_pad / 16};
    s.bytes       = c.used;
    return s;
}

struct BackwardSpace
{
    float *bias, *sums, *parts;
    Panel xr, xt, wr, wt, dr, dt;
    size_t bytes;
};

BackwardSpace backward_space(char *base, const Plan &p, int64_t N, int64_t K)
{
    BackwardSpace s;
    Carver c{base};
    const int64_t v_pad = padded(p.v_piece);
    s.bias  = c.take<float>((size_t)v_pad * 4);
    s.sums  = c.take<float>((size_t)(p.n_pad / 32 * v_pad) * 4);
    s.parts = c.take<float>(p.gx.splits > 1 ? (size_t)p.gx.splits * (size_t)(N * K) * 4 : 0);
    s.xr    = Panel{c.take<char>((size_t)panel_bytes(p.n_pad, p.k_pad)), p.k_pad / 16};
    s.xt    = Panel{c.take<char>((size_t)panel_bytes(p.k_pad, p.n_pad)), p.n_pad / 16};
    s.wr    = Panel{c.take<char>((size_t)panel_bytes(v_pad, p.k_pad)), p.k_pad / 16};
    s.wt    = Panel{c.take<char>((size_t)panel_bytes(p.k_pad, v_pad)), v_pad / 16};
    s.dr    = Panel{c.take<char>((size_t)panel_bytes(v_pad, p.n_pad)), p.n_pad / 16};
    s.dt    = Panel{c.take<char>((size_t)panel_bytes(p.n_pad, v_pad)), v_pad / 16};
    s.bytes = c.used;
    return s;
}

// Sizes the kernels index with: an operand's tile of 256 rows must be reachable with 31-bit byte offsets.
constexpr int64_t kMostRows = (int64_t)1 << 20, kMostVocabulary = (int64_t)1 << 30;

int check_sizes(const char *who, int64_t N, int64_t K, int64_t V)
{
    ODL_REQUIRE(N >= 0 && K > 0 && V > 0, "%s: needs N >= 0, K > 0 and V > 0, got N=%lld K=%lld V=%lld", who, (long long)N, (long long)K, (long long)V);
    ODL_REQUIRE(N <= kMostRows && K <= kMostRows && V <= kMostVocabulary, "%s: N and K up to %lld, V up to %lld, got N=%lld K=%lld V=%lld", who,
                (long long)kMostRows, (long long)kMostVocabulary, (long long)N, (long long)K, (long long)V);
    return ODL_OK;
}

GemmArgs product(const Panel &a, const Panel &b, int64_t contraction)
{
    GemmArgs g{};
    g.a = a, g.b = b, g.nkb = contraction_blocks(contraction), g.batch = 1;
    return g;
}

__global__ void ce_empty_kernel(float *saved)
{
    if (threadIdx.x < kSavedWords)
        saved[threadIdx.x] = threadIdx.x == kScaleX || threadIdx.x == kScaleW ? 1.f : 0.f;
}
}  // namespace

namespace odl
{
namespace linear_ce
{
size_t join_scratch_bytes(int64_t N)
{
    return (size_t)ceil_div(N, kJoinRows) * 16;
}

int join(const float *part_m, const float *part_s, const float *target, int64_t tiles, int64_t n_pad, const Labels &labels, float *row_stats, void *scratch,
         float *saved, hipStream_t st)
{
    const int64_t blocks = ceil_div(labels.N, kJoinRows);
    double *block_loss   = static_cast<double *>(scratch);
    ce_join_kernel<<<dim3((unsigned)blocks), dim3(kBlock), 0, st>>>(part_m, part_s, target, tiles, n_pad, labels, row_stats, block_loss,
                                                                    reinterpret_cast<int *>(block_loss + blocks), saved);
    ODL_LAUNCH_CHECK();
    return ODL_OK;
}
}  // namespace linear_ce
}  // namespace odl

extern "C" size_t odl_hip_linear_softmax_ce_forward_workspace_bytes(int64_t N, int64_t K, int64_t V)
{
    if (N <= 0 || K <= 0 || V <= 0 || N > kMostRows || K > kMostRows || V > kMostVocabulary)
        return 0;
    if (few_rows(N, K, V))
        return few_forward_bytes(N, K, V);
    return forward_space(nullptr, make_plan(N, K, V, false), N, K, V).bytes;
}

extern "C" size_t odl_hip_linear_softmax_ce_row_stats_floats(int64_t N, int64_t K, int64_t V)
{
    if (N <= 0 || K <= 0 || V <= 0 || N > kMostRows || K > kMostRows || V > kMostVocabulary)
        return 0;
    return (size_t)(2 * N) + (few_rows(N, K, V) ? few_kept_floats(N, K, V) : 0);
}

extern "C" size_t odl_hip_linear_softmax_ce_backward_workspace_bytes(int64_t N, int64_t K, int64_t V)
{
    if (N <= 0 || K <= 0 || V <= 0 || N > kMostRows || K > kMostRows || V > kMostVocabulary)
        return 0;
    if (few_rows(N, K, V))
        return few_backward_bytes(N, K, V);
    return backward_space(nullptr, make_plan(N, K, V, true), N, K).bytes;
}

extern "C" int odl_hip_linear_softmax_ce_forward(const float *x, const float *w, int w_out_in, const float *b, const void *t, int idx_is_i64,
                                                 int64_t ignore_index, int64_t N, int64_t K, int64_t V, float *saved8, float *row_stats,
                                                 void *workspace, size_t workspace_bytes, void *stream)
{
    const char *who = "linear_softmax_ce_forward";
    if (int rc = check_sizes(who, N, K, V))
        return rc;
    ODL_REQUIRE(saved8, "%s: null output", who);
    ODL_REQUIRE(N == 0 || (x && w && t && row_stats), "%s: null argument", who);
    hipStream_t st = odl::as_stream(stream);
    if (N == 0)
    {
        ODL_REQUIRE_DEVICE();
        ce_empty_kernel<<<dim3(1), dim3(64), 0, st>>>(saved8);
        ODL_LAUNCH_CHECK();
        return ODL_OK;
    }
    const size_t need = odl_hip_linear_softmax_ce_forward_workspace_bytes(N, K, V);
    ODL_REQUIRE(workspace && workspace_bytes >= need, "%s: workspace of %zu bytes needed, got %zu", who, need, workspace ? workspace_bytes : (size_t)0);
    ODL_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "%s: the workspace must be 16-byte aligned", who);
    ODL_REQUIRE_DEVICE();
    if (few_rows(N, K, V))
        return few_forward(Problem{x, w, b, w_out_in, Labels{t, idx_is_i64, ignore_index, V, N}, N, K, V}, saved8, row_stats, static_cast<char *>(workspace), st);
    const Plan p = make_plan(N, K, V, false);
    const ForwardSpace s = forward_space(static_cast<char *>(workspace), p, N, K, V);
    const Labels labels{t, idx_is_i64, ignore_index, V, N};
    const int mx = magnitude_blocks(N * K), mw = magnitude_blocks(K * V);
    ce_magnitudes_kernel<<<dim3(mx + mw), dim3(kBlock), 0, st>>>(x, N, K, labels, w, K * V, mx, s.mags, saved8);
    ODL_LAUNCH_CHECK();
    int64_t tiles_done = 0;
    for (int64_t i = 0; i < p.pieces; ++i)
    {
        const int64_t vn = p.vn(V, i), v_pad = padded(vn);
        PrepArgs a{};
        a.x = x, a.w = w, a.b = b, a.N = N, a.K = K, a.V = V, a.w_out_in = w_out_in, a.v0 = i * p.v_piece, a.vn = vn;
        a.xr = s.xr, a.wr = s.wr, a.bias = s.bias, a.labels = labels, a.mags = i == 0 ? s.mags : nullptr, a.mags_x = mx, a.mags_w = mw, a.saved = saved8;
        a.x_tiles_r = i == 0 ? (int)(p.n_pad / 64) : 0, a.x_tiles_c = (int)(p.k_pad / 64);
        a.w_tiles_r = (int)((w_out_in ? v_pad : p.k_pad) / 64), a.w_tiles_c = (int)((w_out_in ? p.k_pad : v_pad) / 64);
        a.bias_blocks = (int)odl::ceil_div(v_pad, kBlock);
        ce_prepare_kernel<<<dim3((unsigned)(a.x_tiles_r * a.x_tiles_c + a.w_tiles_r * a.w_tiles_c + a.bias_blocks)), dim3(kBlock), 0, st>>>(a);
        ODL_LAUNCH_CHECK();
        const Cut cut = pick_cut(v_pad, p.n_pad, false, 1, contraction_blocks(K));
        const StatsEpilogue e{s.bias, saved8, labels, a.v0, p.n_pad, s.part_m + tiles_done * p.n_pad, s.part_s + tiles_done * p.n_pad, s.target};
        if (int rc = launch_gemm(product(s.wr, s.xr, K), v_pad, p.n_pad, cut, e, st))
            return rc;
        tiles_done += v_pad / cut.bm;
    }
    return join(s.part_m, s.part_s, s.target, tiles_done, p.n_pad, labels, row_stats, s.join_scratch, saved8, st);
}

extern "C" int odl_hip_linear_softmax_ce_backward(const float *device_gy, const float *x, const float *w, int w_out_in, const float *b, const void *t,
                                                  int idx_is_i64, int64_t ignore_index, int64_t N, int64_t K, int64_t V, const float *saved8,
                                                  const float *row_stats, float *gx, float *gw, float *gb, void *workspace, size_t workspace_bytes,
                                                  void *stream)
{
    const char *who = "linear_softmax_ce_backward";
    if (int rc = check_sizes(who, N, K, V))
        return rc;
    ODL_REQUIRE(saved8, "%s: null argument", who);
    ODL_REQUIRE(N == 0 || (x && w && t && row_stats), "%s: null argument", who);
    hipStream_t st = odl::as_stream(stream);
    if (!gx && !gw && !gb)
        return ODL_OK;
    if (N == 0)
    {
        ODL_REQUIRE_DEVICE();
        if (gw)
            if (int rc = odl::fill_launch(gw, K * V, 0.f, st))
                return rc;
        if (gb)
            if (int rc = odl::fill_launch(gb, V, 0.f, st))
                return rc;
        return ODL_OK;
    }
    const size_t need = odl_hip_linear_softmax_ce_backward_workspace_bytes(N, K, V);
    ODL_REQUIRE(workspace && workspace_bytes >= need, "%s: workspace of %zu bytes needed, got %zu", who, need, workspace ? workspace_bytes : (size_t)0);
    ODL_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "%s: the workspace must be 16-byte aligned", who);
    ODL_REQUIRE_DEVICE();
    if (few_rows(N, K, V))
        return few_backward(Problem{x, w, b, w_out_in, Labels{t, idx_is_i64, ignore_index, V, N}, N, K, V}, device_gy, saved8, row_stats, gx, gw, gb,
                            static_cast<char *>(workspace), st);
    const Plan p = make_plan(N, K, V, true);
    const BackwardSpace s = backward_space(static_cast<char *>(workspace), p, N, K);
    const Labels labels{t, idx_is_i64, ignore_index, V, N};
    for (int64_t i = 0; i < p.pieces; ++i)
    {
        const int64_t v0 = i * p.v_piece, vn = p.vn(V, i), v_pad = padded(vn);
        PrepArgs a{};
        a.x = x, a.w = w, a.b = b, a.N = N, a.K = K, a.V = V, a.w_out_in = w_out_in, a.v0 = v0, a.vn = vn;
        a.xr = s.xr, a.wr = s.wr, a.bias = s.bias, a.labels = labels, a.saved = const_cast<float *>(saved8);
        if (gw)
            a.xt = s.xt;
        if (gx)
            a.wt = s.wt;
        a.x_tiles_r = i == 0 ? (int)(p.n_pad / 64) : 0, a.x_tiles_c = (int)(p.k_pad / 64);
        a.w_tiles_r = (int)((w_out_in ? v_pad : p.k_pad) / 64), a.w_tiles_c = (int)((w_out_in ? p.k_pad : v_pad) / 64);
        a.bias_blocks = (int)odl::ceil_div(v_pad, kBlock);
        ce_prepare_kernel<<<dim3((unsigned)(a.x_tiles_r * a.x_tiles_c + a.w_tiles_r * a.w_tiles_c + a.bias_blocks)), dim3(kBlock), 0, st>>>(a);
        ODL_LAUNCH_CHECK();
        const Cut cut = pick_cut(v_pad, p.n_pad, false, 1, contraction_blocks(K));
        GradEpilogue e{s.bias, saved8, row_stats, labels, v0, Panel{nullptr, 0}, Panel{nullptr, 0}, gb ? s.sums : nullptr, v_pad};
        if (gx)
            e.dt = s.dt;
        if (gw)
            e.dr = s.dr;
        if (int rc = launch_gemm(product(s.wr, s.xr, K), v_pad, p.n_pad, cut, e, st))
            return rc;
        if (gw)
        {
            // [V, K]: rows of vocabulary; [K, V]: rows of K, so that lanes run along the stored rows either way
            const OutEpilogue o = w_out_in ? OutEpilogue{gw + v0 * K, vn, K, K, 0, saved8, kScaleX, device_gy, 0}
                                           : OutEpilogue{gw + v0, K, vn, V, 0, saved8, kScaleX, device_gy, 0};
            const int64_t rows = w_out_in ? v_pad : p.k_pad, cols = w_out_in ? p.k_pad : v_pad;
            if (int rc = launch_gemm(w_out_in ? product(s.dr, s.xt, N) : product(s.xt, s.dr, N), rows, cols, pick_cut(rows, cols, false, 1, contraction_blocks(N)), o, st))
                return rc;
        }
        if (gx)
        {
            // a shorter last piece keeps the runs' length: those past its end have nothing to add
            Cut gx_cut       = p.gx;
            const int nkb    = contraction_blocks(vn);
            gx_cut.split_kb  = std::min(gx_cut.split_kb, nkb);
            gx_cut.splits    = (int)odl::ceil_div(nkb, gx_cut.split_kb);
            const OutEpilogue o{p.gx.splits > 1 ? s.parts : gx, N, K, K, N * K, saved8, kScaleW, device_gy, i > 0};
            if (int rc = launch_gemm(product(s.dt, s.wt, vn), p.n_pad, p.k_pad, gx_cut, o, st))
                return rc;
        }
        const int64_t n            = N * K;
        const unsigned bias_blocks = gb ? (unsigned)(v_pad / 64) : 0u;
        const unsigned gx_blocks   = gx && p.gx.splits > 1 && i + 1 == p.pieces ? (unsigned)std::min<int64_t>(2048, odl::ceil_div(n, kBlock)) : 0u;
        if (bias_blocks + gx_blocks)
        {
            const int waves_n = cut.bn == 256 ? 4 : 2;
            const BiasGrad bias{s.sums, (int)(p.n_pad / cut.bn) * waves_n, v_pad, vn, gb ? gb + v0 : nullptr, saved8, device_gy};
            ce_sums_kernel<<<dim3(bias_blocks + gx_blocks), dim3(kBlock), 0, st>>>(bias, bias_blocks, s.parts, p.gx.splits, n, gx);
            ODL_LAUNCH_CHECK();
        }
    }
    return ODL_OK;
}
