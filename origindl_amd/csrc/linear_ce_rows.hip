// The output layer with its loss for up to 64 rows: scoring a few positions, small batches.
//
// What bounds it: the bytes of w. A pass over w [V, K] multiplies 2N operations per element of 4 bytes, which the float32 matrix
// instructions do in less time than memory delivers w (N = 64: as fast). So nothing is laid out first: w streams once from
// where it lies into float32 matrix instructions (v_mfma_f32_32x32x2), per pass:
//   forward    one pass: logits of 128 entries a workgroup, their maximum and sum of powers in its epilogue
//   backward   one pass for the logits again, whose epilogue writes d = softmax - one-hot ([V][N] floats: the weights' size
//              times N / K) and gb; one pass for gx = d.w, in runs of the vocabulary; gw = d^T.x writes its size once.
//
// Both products with w are one kernel: w is [out][contraction] for the logits of a [V, K] weight and [contraction][out] for its
// gx, and the other way round for a [K, V] weight. Eight waves share a tile of 128 outputs, each takes an eighth of the
// contraction, 8 values a step: lanes of the lower half-wave the first four, of the upper half the others, so that w and the
// small operand both arrive as 16 bytes a lane. The small operand lies as q[contraction / 4][rows][4], zeros past the ends and
// in rows that do not count.
#include <algorithm>

#include "linear_ce.h"

namespace
{
using namespace odl::linear_ce;
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));  // rows of w need not start on 16 bytes

constexpr int kWaves = 8, kTile = 128;

// x as q[k / 4][rows][4]; rows = 32 or 64. Also clears the ticket of the joining launch.
__global__ __launch_bounds__(kBlock) void ce_rows_prepare_kernel(const float *__restrict__ x, int64_t K, const Labels labels, int rows, int64_t quads,
                                                                 f32x4 *__restrict__ q, float *saved)
{
    if (saved && blockIdx.x == 0 && threadIdx.x == 0)
        reinterpret_cast<int *>(saved)[kTicket] = 0;
    const int64_t at = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (at >= quads * rows)
        return;
    // consecutive threads take consecutive quads of one row: x is read in whole lines
    const int64_t n = at / quads, kq = at - n * quads;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (labels(n) >= 0)
    {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (kq * 4 + e < K)
                v[e] = x[n * K + kq * 4 + e];
    }
    q[kq * rows + n] = v;
}

struct Stream
{
    const float *w;
    int64_t ld, outs, contraction;
    const f32x4 *q;      // [groups * 2][NB * 32]
    int64_t groups;      // steps of 8 contraction values
    int64_t wave_groups; // steps of one wave
};

// OUT_ROWS: w is [out][contraction], else [contraction][out]. The epilogue is called by the first four waves with block m of
// the tile: element 4q + e of s[nb] is row 8q + 4 * (lane / 32) + e of the block, column nb * 32 + lane % 32; a block's row r
// is output 32m + r of the tile (OUT_ROWS) or 4r + m.
template <int NB, bool OUT_ROWS, class Epilogue>
__global__ __launch_bounds__(64 * kWaves, 2) void ce_stream_kernel(const Stream a, const Epilogue epilogue)
{
    __shared__ f32x4 lds[kWaves * 4 * 256];
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31;
    const int64_t o0 = (int64_t)blockIdx.x * kTile;
    f32x16 acc[4][NB];
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                acc[m][nb][e] = 0.f;
    struct Step
    {
        f32x4 w[4], q[NB];
    };
    const f32x4 *q = a.q + (int64_t)half * NB * 32 + col;
    const int64_t first = ((int64_t)blockIdx.y * kWaves + wave) * a.wave_groups, last = min(first + a.wave_groups, a.groups);
    const int64_t whole = a.outs >= 4 || OUT_ROWS ? min(last, a.contraction / 8) : first;
    // In the last tile a lane past the outputs reads what lies in reach instead (its outputs are nobody's); of four outputs that
    // straddle the end it reads the last four and moves them to their places.
    const int64_t o_lane = o0 + col * 4, shift = OUT_ROWS ? 0 : o_lane + 4 - a.outs;
    const float *w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] = OUT_ROWS ? a.w + min(o0 + 32 * i + col, a.outs - 1) * a.ld + half * 4 : a.w + (int64_t)(half * 4 + i) * a.ld + (shift > 0 ? a.outs - 4 : o_lane);
    const int64_t w_step = OUT_ROWS ? 8 : 8 * a.ld;
    const auto load = [&](int64_t g, Step &s) {
        const int64_t at = min(g, whole - 1);  // past the wave's last whole step: that one again, multiplied by nobody
#pragma unroll
        for (int i = 0; i < 4; ++i)
            s.w[i] = *reinterpret_cast<const f32x4u *>(w[i] + at * w_step);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
            s.q[nb] = q[at * 2 * NB * 32 + nb * 32];
    };
    // the contraction's last values, single loads with zeros past its end (and outputs fewer than four)
    const auto load_guarded = [&](int64_t g, Step &s) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
            s.q[nb] = q[g * 2 * NB * 32 + nb * 32];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
            {
                const int64_t o = OUT_ROWS ? o0 + 32 * i + col : o0 + col * 4 + e, c = g * 8 + half * 4 + (OUT_ROWS ? e : i);
                s.w[i][e] = o < a.outs && c < a.contraction ? a.w[OUT_ROWS ? o * a.ld + c : c * a.ld + o] : 0.f;
            }
    };
    const bool straddles = !OUT_ROWS && o0 + kTile > a.outs;
    const auto multiply = [&](const Step &s, bool move) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
        {
            f32x4 v = s.w[j];
            if (move)
            {
                v = shift == 1 ? f32x4{v[1], v[2], v[3], 0.f} : v;
                v = shift == 2 ? f32x4{v[2], v[3], 0.f, 0.f} : v;
                v = shift == 3 ? f32x4{v[3], 0.f, 0.f, 0.f} : v;
            }
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
                    acc[m][nb] = __builtin_amdgcn_mfma_f32_32x32x2f32(OUT_ROWS ? s.w[m][j] : v[m], s.q[nb][j], acc[m][nb], 0, 0, 0);
        }
    };
    if (first < whole)
    {
        Step s0, s1, t0, t1;
        load(first, s0), load(first + 1, s1);
        for (int64_t g = first; g < whole; g += 4)
        {
            load(g + 2, t0), load(g + 3, t1);
            multiply(s0, straddles);
            if (g + 1 < whole)
                multiply(s1, straddles);
            load(g + 4, s0), load(g + 5, s1);
            if (g + 2 < whole)
                multiply(t0, straddles);
            if (g + 3 < whole)
                multiply(t1, straddles);
        }
    }
    for (int64_t g = max(first, whole); g < last; ++g)
    {
        Step s;
        load_guarded(g, s);
        multiply(s, false);
    }
    // the waves' sums, one block of columns at a time; wave m < 4 adds up block m in the waves' order
    f32x16 sum[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
    {
        if (nb)
            __syncthreads();
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                lds[(wave * 4 + m) * 256 + i * 64 + lane] = f32x4{acc[m][nb][4 * i], acc[m][nb][4 * i + 1], acc[m][nb][4 * i + 2], acc[m][nb][4 * i + 3]};
        __syncthreads();
        if (wave < 4)
        {
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
                f32x4 v = lds[wave * 256 + i * 64 + lane];
#pragma unroll
                for (int w = 1; w < kWaves; ++w)
                    v += lds[(w * 4 + wave) * 256 + i * 64 + lane];
                sum[nb][4 * i] = v[0], sum[nb][4 * i + 1] = v[1], sum[nb][4 * i + 2] = v[2], sum[nb][4 * i + 3] = v[3];
            }
        }
    }
    __syncthreads();  // the epilogue writes LDS
    epilogue.template run<NB, OUT_ROWS>(o0, wave, lane, sum, reinterpret_cast<float *>(lds));
}

// output (vocabulary entry, or feature) of element e of a lane's block m
template <bool OUT_ROWS>
__device__ inline int64_t output_of(int64_t o0, int m, int lane, int e)
{
    const int r = 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
    return o0 + (OUT_ROWS ? 32 * m + r : 4 * r + m);
}

struct RowsStatsEpilogue
{
    const float *b;
    Labels labels;
    int64_t V, n_pad;
    float *part_m, *part_s, *target;
    template <int NB, bool OUT_ROWS>
    __device__ void run(int64_t o0, int m, int lane, f32x16 *z, float *lds) const
    {
        float *lm = lds, *ls = lds + 4 * NB * 32;
        if (m < 4)
        {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
            {
                const int64_t n = nb * 32 + (lane & 31), label = labels(n);
                float top = -INFINITY;
#pragma unroll
                for (int e = 0; e < 16; ++e)
                {
                    const int64_t v = output_of<OUT_ROWS>(o0, m, lane, e);
                    z[nb][e] = v < V ? z[nb][e] + (b ? b[v] : 0.f) : -INFINITY;
                    if (v == label)
                        target[n] = z[nb][e];
                    top = fmaxf(top, z[nb][e]);
                }
                float m2 = top * kLog2e, s = 0.f;
                const float sub = finite_top(m2);
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    s += pow2(fmaf(z[nb][e], kLog2e, -sub));
                const float m_o = __shfl_xor(m2, 32, 64), s_o = __shfl_xor(s, 32, 64);
                merge(m2, s, m_o, s_o);
                if (lane < 32)
                    lm[m * NB * 32 + nb * 32 + lane] = m2, ls[m * NB * 32 + nb * 32 + lane] = s;
            }
        }
        __syncthreads();
        if (threadIdx.x < NB * 32)
        {
            const int n = threadIdx.x;
            float m2 = lm[n], s = ls[n];
#pragma unroll
            for (int i = 1; i < 4; ++i)
                merge(m2, s, lm[i * NB * 32 + n], ls[i * NB * 32 + n]);
            part_m[(int64_t)blockIdx.x * n_pad + n] = m2, part_s[(int64_t)blockIdx.x * n_pad + n] = s;
        }
    }
};

// d in the small operand's layout, dq[v / 4][rows][4], and gb
struct RowsGradEpilogue
{
    const float *b, *saved, *row, *gy;
    Labels labels;
    int64_t V;
    float *dq, *gb;
    template <int NB, bool OUT_ROWS>
    __device__ void run(int64_t o0, int m, int lane, f32x16 *z, float *) const
    {
        if (m >= 4)
            return;
        float sums[16];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
        {
            const int64_t n = nb * 32 + (lane & 31), label = labels(n);
            const bool counts = label >= 0;
            const float m2 = counts ? row[2 * n] : 0.f, inv = counts ? 1.f / row[2 * n + 1] : 0.f;
#pragma unroll
            for (int e = 0; e < 16; ++e)
            {
                const int64_t v = output_of<OUT_ROWS>(o0, m, lane, e);
                float d = 0.f;
                if (counts && v < V)
                {
                    const float logit = z[nb][e] + (b ? b[v] : 0.f);
                    d = pow2(fmaf(logit, kLog2e, -m2)) * inv;
                    if (v == label)
                        d -= 1.f;
                }
                z[nb][e] = d;
                sums[e]  = nb ? sums[e] + d : d;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
                if constexpr (OUT_ROWS)
                    *reinterpret_cast<f32x4 *>(dq + ((output_of<true>(o0, m, lane, 4 * i) / 4) * NB * 32 + n) * 4) =
                        f32x4{z[nb][4 * i], z[nb][4 * i + 1], z[nb][4 * i + 2], z[nb][4 * i + 3]};
                else
                {
#pragma unroll
                    for (int e = 4 * i; e < 4 * i + 4; ++e)
                        dq[((output_of<false>(o0, m, lane, e) / 4) * NB * 32 + n) * 4 + m] = z[nb][e];
                }
            }
        }
        if (!gb)
            return;
        const float g = (gy ? *gy : 1.f) / fmaxf(saved[kCounted], 1.f);
#pragma unroll
        for (int e = 0; e < 16; ++e)
        {
            float s = sums[e];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1)
                s += __shfl_xor(s, o, 64);
            const int64_t v = output_of<OUT_ROWS>(o0, m, lane, e);
            if ((lane & 31) == 0 && v < V)
                gb[v] = s * g;
        }
    }
};

// parts[run][feature][rows]
struct RowsPartEpilogue
{
    float *parts;
    int64_t outs;
    template <int NB, bool OUT_ROWS>
    __device__ void run(int64_t o0, int m, int lane, f32x16 *z, float *) const
    {
        if (m >= 4)
            return;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int e = 0; e < 16; ++e)
            {
                const int64_t o = output_of<OUT_ROWS>(o0, m, lane, e);
                if (o < outs)
                    parts[((int64_t)blockIdx.y * outs + o) * NB * 32 + nb * 32 + (lane & 31)] = z[nb][e];
            }
    }
};

// gx[n][k] = factor * the runs' sums, in order; a workgroup takes 32 features
__global__ __launch_bounds__(kBlock) void ce_rows_gx_kernel(const float *__restrict__ parts, int runs, int64_t N, int64_t K, int rows, const float *saved, const float *gy,
                                                            float *__restrict__ gx)
{
    __shared__ float tile[32][65];
    const float g = (gy ? *gy : 1.f) / fmaxf(saved[kCounted], 1.f);
    const int64_t k0 = (int64_t)blockIdx.x * 32;
    for (int i = threadIdx.x; i < 32 * rows; i += kBlock)
    {
        const int k = i / rows, n = i % rows;
        float s = 0.f;
        if (k0 + k < K)
#pragma unroll 8
            for (int r = 0; r < runs; ++r)
                s += parts[((int64_t)r * K + k0 + k) * rows + n];
        tile[k][n] = s * g;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * rows; i += kBlock)
    {
        const int n = i / 32, k = i % 32;
        if (n < N && k0 + k < K)
            gx[n * K + k0 + k] = tile[k][n];
    }
}

// gw = factor * d^T.x over NB * 32 rows. out[r][c]: qc the operand of the stored rows' direction (16 bytes a lane: four columns),
// qr the other one's. A wave keeps its 128 columns' operand in registers and walks down `steps` blocks of 32 rows.
template <int NB>
__global__ __launch_bounds__(kBlock) void ce_rows_outer_kernel(const f32x4 *__restrict__ qc, const float *__restrict__ qr, int64_t rows, int64_t cols, unsigned tiles_c, int steps,
                                                               const float *saved, const float *gy, float *__restrict__ out)
{
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, half = lane >> 5, i32 = lane & 31;
    const float g = (gy ? *gy : 1.f) / fmaxf(saved[kCounted], 1.f);
    const unsigned group = blockIdx.x / tiles_c;
    const int64_t c0 = (int64_t)(blockIdx.x - group * tiles_c) * 128;
    f32x4 c[NB * 16];
#pragma unroll
    for (int i = 0; i < NB * 16; ++i)
        c[i] = qc[(c0 / 4 + i32) * NB * 32 + 2 * i + half];
    const int64_t col = c0 + i32 * 4;
    for (int step = 0; step < steps; ++step)
    {
        const int64_t r0 = (((int64_t)group * steps + step) * 4 + wave) * 32;
        if (r0 >= rows)
            return;
        const float *q = qr + ((r0 + i32) / 4) * NB * 32 * 4 + (i32 & 3);
        f32x16 acc[4];
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                acc[m][e] = 0.f;
        float r[NB * 16];
#pragma unroll
        for (int i = 0; i < NB * 16; ++i)
            r[i] = q[(2 * i + half) * 4];
#pragma unroll
        for (int i = 0; i < NB * 16; ++i)
#pragma unroll
            for (int m = 0; m < 4; ++m)
                acc[m] = __builtin_amdgcn_mfma_f32_32x32x2f32(r[i], c[i][m], acc[m], 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 16; ++e)
        {
            const int64_t row = r0 + 8 * (e >> 2) + 4 * half + (e & 3);
            if (row >= rows)
                continue;
            float *at = out + row * cols + col;
            if (col + 3 < cols)
                *reinterpret_cast<f32x4u *>(at) = f32x4{acc[0][e] * g, acc[1][e] * g, acc[2][e] * g, acc[3][e] * g};
            else
            {
#pragma unroll
                for (int m = 0; m < 4; ++m)
                    if (col + m < cols)
                        at[m] = acc[m][e] * g;
            }
        }
    }
}

int rows_of(int64_t N)
{
    return N <= 32 ? 32 : 64;
}

// quads of a small operand: whole tiles of 128, so that a tile of gw reads only what exists
int64_t quads_of(int64_t n)
{
    return odl::ceil_div(n, 128) * 32;
}

int runs_for_gx(int64_t K, int64_t V)
{
    const int64_t tiles = odl::ceil_div(K, kTile);
    return (int)std::max<int64_t>(1, std::min<int64_t>(odl::device_cus() / tiles, odl::ceil_div(V, 128)));
}

struct FewSpace
{
    f32x4 *xq;
    float *part_m, *part_s, *target, *dq, *parts;
    void *join_scratch;
    size_t bytes;
};

FewSpace forward_space(char *base, int64_t N, int64_t K, int64_t V)
{
    FewSpace s{};
    Carver c{base};
    const size_t rows = (size_t)rows_of(N), tiles = (size_t)odl::ceil_div(V, kTile);
    s.xq           = c.take<f32x4>((size_t)quads_of(K) * rows * 16);
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
    const size_t rows = (size_t)rows_of(N);
    s.xq    = c.take<f32x4>((size_t)quads_of(K) * rows * 16);
    s.dq    = c.take<float>((size_t)quads_of(V) * rows * 16);
    s.parts = c.take<float>((size_t)runs_for_gx(K, V) * (size_t)K * rows * 4);
    s.bytes = c.used;
    return s;
}

template <class Epilogue>
int stream(const float *w, bool out_rows, int64_t ld, int64_t outs, int64_t contraction, const void *q, int rows, int runs, const Epilogue &e, hipStream_t st)
{
    Stream a{w, ld, outs, contraction, static_cast<const f32x4 *>(q), odl::ceil_div(contraction, 8), 0};
    a.wave_groups = odl::ceil_div(a.groups, (int64_t)runs * kWaves);
    const dim3 grid((unsigned)odl::ceil_div(outs, kTile), (unsigned)runs), block(64 * kWaves);
    if (rows == 32 && out_rows)
        ce_stream_kernel<1, true, Epilogue><<<grid, block, 0, st>>>(a, e);
    else if (rows == 32)
        ce_stream_kernel<1, false, Epilogue><<<grid, block, 0, st>>>(a, e);
    else if (out_rows)
        ce_stream_kernel<2, true, Epilogue><<<grid, block, 0, st>>>(a, e);
    else
        ce_stream_kernel<2, false, Epilogue><<<grid, block, 0, st>>>(a, e);
    ODL_LAUNCH_CHECK();
    return ODL_OK;
}

int prepare(const Problem &p, int rows, f32x4 *xq, float *saved, hipStream_t st)
{
    const int64_t quads = quads_of(p.K);
    ce_rows_prepare_kernel<<<dim3((unsigned)odl::ceil_div(quads * rows, kBlock)), dim3(kBlock), 0, st>>>(p.x, p.K, p.labels, rows, quads, xq, saved);
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

int few_forward(const Problem &p, float *saved, float *row_stats, char *workspace, hipStream_t st)
{
    const int rows = rows_of(p.N);
    const FewSpace s = ::forward_space(workspace, p.N, p.K, p.V);
    if (int rc = prepare(p, rows, s.xq, saved, st))
        return rc;
    const RowsStatsEpilogue e{p.b, p.labels, p.V, rows, s.part_m, s.part_s, s.target};
    if (int rc = stream(p.w, p.w_out_in != 0, p.w_out_in ? p.K : p.V, p.V, p.K, s.xq, rows, 1, e, st))
        return rc;
    return join(s.part_m, s.part_s, s.target, ceil_div(p.V, kTile), rows, p.labels, row_stats, s.join_scratch, saved, st);
}

int few_backward(const Problem &p, const float *gy, const float *saved, const float *row_stats, float *gx, float *gw, float *gb, char *workspace,
                 hipStream_t st)
{
    const int rows = rows_of(p.N);
    const FewSpace s = ::backward_space(workspace, p.N, p.K, p.V);
    if (int rc = prepare(p, rows, s.xq, nullptr, st))
        return rc;
    const int64_t ld = p.w_out_in ? p.K : p.V;
    const RowsGradEpilogue e{p.b, saved, row_stats, gy, p.labels, p.V, s.dq, gb};
    if (int rc = stream(p.w, p.w_out_in != 0, ld, p.V, p.K, s.xq, rows, 1, e, st))
        return rc;
    if (gx)
    {
        const int runs = runs_for_gx(p.K, p.V);
        if (int rc = stream(p.w, p.w_out_in == 0, ld, p.K, p.V, s.dq, rows, runs, RowsPartEpilogue{s.parts, p.K}, st))
            return rc;
        ce_rows_gx_kernel<<<dim3((unsigned)ceil_div(p.K, 32)), dim3(kBlock), 0, st>>>(s.parts, runs, p.N, p.K, rows, saved, gy, gx);
        ODL_LAUNCH_CHECK();
    }
    if (gw)
    {
        const int64_t r = p.w_out_in ? p.V : p.K, c = p.w_out_in ? p.K : p.V;
        const void *qc = p.w_out_in ? (const void *)s.xq : s.dq, *qr = p.w_out_in ? (const void *)s.dq : s.xq;
        // enough workgroups for the chip, and as many rows each as that leaves: the columns' operand is read once per workgroup
        const int64_t tiles_c = ceil_div(c, 128), tiles_r = ceil_div(r, 128);
        const int steps = (int)std::max<int64_t>(1, std::min<int64_t>(16, tiles_c * tiles_r / (8 * (int64_t)device_cus())));
        const int64_t blocks = tiles_c * ceil_div(tiles_r, steps);
        ODL_REQUIRE(blocks < ((int64_t)1 << 31), "weight gradient of too many tiles");
        const dim3 grid((unsigned)blocks);
        if (rows == 32)
            ce_rows_outer_kernel<1><<<grid, dim3(kBlock), 0, st>>>(static_cast<const f32x4 *>(qc), static_cast<const float *>(qr), r, c, (unsigned)tiles_c, steps, saved, gy, gw);
        else
            ce_rows_outer_kernel<2><<<grid, dim3(kBlock), 0, st>>>(static_cast<const f32x4 *>(qc), static_cast<const float *>(qr), r, c, (unsigned)tiles_c, steps, saved, gy, gw);
        ODL_LAUNCH_CHECK();
    }
    return ODL_OK;
}
}  // namespace linear_ce
}  // namespace odl
