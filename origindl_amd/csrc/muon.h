// What the two implementations of the orthogonalised update share: muon.hip (any matrix) and muon_slim.hip (a short side up to
// 128).
#pragma once
#include "split_gemm.h"

namespace odl
{
namespace muon
{
using namespace odl::split;

constexpr int kBlock     = 256;
constexpr float kScale   = 8192.f;
constexpr double kMost   = 7.5;
constexpr int kGroup     = 32;  // matrices per launch

struct Matrices  // one launch's matrices: all [rows, cols]
{
    const float *g[kGroup];
    float *buf[kGroup];    // null: U is the gradient itself
    const float *p[kGroup];
    float *out[kGroup];    // X, or the new parameter where p is not null
    float rate[kGroup];    // what X is multiplied by before it is taken from the parameter
    int64_t rows, cols;
    float momentum;
    int nesterov;

};

// U's element i; buf holds the new momentum already
struct Update
{
    const float *g, *buf;
    float momentum;
    int nesterov;
    __device__ float operator()(int64_t i) const
    {
        if (!buf)
            return g[i];
        return nesterov ? g[i] + momentum * buf[i] : buf[i];
    }
};

struct UpdateAt
{
    Update u;
    int64_t cols;
    __device__ float operator()(int64_t r, int64_t c) const { return u(r * cols + c); }
};

// the accumulator block as rows of the other side: through the wave's scratch
__device__ inline void store_mirror(const Panel &p, int64_t rb, int64_t cb, int lane, const f32x16 &c, float *scratch)
{
#pragma unroll
    for (int e = 0; e < 16; ++e)
        scratch[(16 * (e >> 3) + 8 * (lane >> 5) + (e & 7)) * 33 + (lane & 31)] = c[e];
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int h = 0; h < 2; ++h)
    {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
            v[e] = scratch[(lane & 31) * 33 + 16 * h + 8 * (lane >> 5) + e];
        store_fragment(p, rb, cb * 2 + h, lane, v);
    }
    __builtin_amdgcn_wave_barrier();
}

// c[8h + e] <- own * acc + before * prev at the block's place in a panel of the column side, kept times kScale
__device__ inline void combine(f32x16 &c, const Panel &prev, int64_t cb, int64_t rb, int lane, float own, float before)
{
#pragma unroll
    for (int h = 0; h < 2; ++h)
    {
        float v[8];
        load_fragment(prev, cb, rb * 2 + h, lane, v);
#pragma unroll
        for (int e = 0; e < 8; ++e)
            c[8 * h + e] = fmaf(own, c[8 * h + e], before * v[e]);
    }
}

__device__ inline void store_columns(const Panel &p, int64_t cb, int64_t rb, int lane, const f32x16 &c)
{
#pragma unroll
    for (int h = 0; h < 2; ++h)
    {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
            v[e] = c[8 * h + e];
        store_fragment(p, cb, rb * 2 + h, lane, v);
    }
}

// a lane's part of X, block (row block rb of m, column block cb of n) of matrix z after to_columns: stored, or applied to the
// parameter
__device__ inline void write_result(const Matrices &a, int z, f32x16 &c, int64_t rb, int64_t cb, int lane, float keep)
{
    const bool tall = a.rows > a.cols;
    const int64_t m = tall ? a.cols : a.rows, n = tall ? a.rows : a.cols, col = cb * 32 + (lane & 31);
    if (col >= n)
        return;
    const int64_t row0 = rb * 32 + 8 * (lane >> 5), at0 = tall ? col * m + row0 : row0 * n + col, step = tall ? 1 : n;
    const float *p = a.p[z], rate = a.rate[z];
    float *out = a.out[z];
    // all of the parameter's elements are under way before the first new one is stored (p may be out)
    if (p)
    {
        float old[16];
#pragma unroll
        for (int e = 0; e < 16; ++e)
        {
            const int row = 16 * (e >> 3) + (e & 7);
            old[e] = row0 + row < m ? p[at0 + row * step] : 0.f;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e)
            c[e] = old[e] * keep - c[e] * rate;
    }
#pragma unroll
    for (int e = 0; e < 16; ++e)
    {
        const int row = 16 * (e >> 3) + (e & 7);
        if (row0 + row < m)
            out[at0 + row * step] = c[e];
    }
}

// the sum of `parts` numbers, in every thread of a workgroup of WAVES waves
template <int WAVES>
__device__ inline double sum_of_parts(const double *sums, int parts, double *scratch)
{
    double s = 0.0;
    for (int i = threadIdx.x; i < parts; i += WAVES * 64)
        s += sums[i];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0)
        scratch[threadIdx.x >> 6] = s;
    __syncthreads();
    s = scratch[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w)
        s += scratch[w];
    return s;
}

// what U is multiplied by to be X0 as an operand; a zero matrix stays one with eps = 0 too
__device__ inline double operand_factor(double squares, double eps)
{
    const double norm = sqrt(squares) + eps;
    return norm == 0.0 ? 0.0 : (double)kScale / norm;
}

// the matrices of one call: rows <= cols on the sides m, n; see muon.hip
struct Settings
{
    int steps;
    float a, b, c, eps, keep;
};

bool slim_fits(int64_t rows, int64_t cols);
bool slim_whole(int64_t rows, int64_t cols);  // slim_run updates the momentum and finds the norm itself
size_t slim_bytes(int64_t rows, int64_t cols);  // of one matrix
// sums: the partial sums of squares of every matrix's update, `parts` of them
int slim_run(const Matrices &mat, int count, const Settings &s, const double *sums, int parts, char *workspace, hipStream_t st);
}  // namespace muon
}  // namespace odl
