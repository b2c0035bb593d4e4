// Newton-Schulz steps on matrices whose short side is at most 128: one launch a step, and one for everything where the long side
// is no longer either.
//
// What bounds it: launches. The products of such a step take a microsecond, a launch that depends on the last one three to
// five. So a workgroup takes a strip of the long side, all m rows of it, and does a whole step: it adds up the strips' shares
// of A = X X^T, forms b A + c A A in LDS (every workgroup for itself: m^3 operations), multiplies it with its strip of X, and
// leaves its strip's share of the next A. Operands are those of split_gemm.h; A and b A + c A A never leave LDS, X's strip is
// updated in place (nobody else reads it), the shares alternate between two places. A matrix of one strip stays in LDS whole.
//
// A matrix of one strip needs no other workgroup: momentum, norm and all steps are one launch (128 x 128, five steps: 53 us, a
// compute unit's matrix instructions being busy for half of it).
//
// Shares are read by every workgroup: strips^2 * m^2 * 2 bytes a step. 64 columns a strip up to 512 columns, 128 above, and up
// to 4096 columns: 1.3 MB a workgroup there, about 8 us.
#include <algorithm>

#include "muon.h"

namespace
{
using namespace odl::muon;

constexpr int64_t kMostM = 128, kMostN = 4096;

struct SlimArgs
{
    Matrices a;
    const double *sums;
    int parts, steps;
    double eps;
    char *xt;  // X by columns: rows of n, contraction m
    int64_t xt_bytes;
    const f32x4 *share_in;
    f32x4 *share_out;
    int strips;
    float ca, cb, cc, keep;
};

enum
{
    kFirst,
    kStep,
    kLast,
    kWhole  // one strip: everything
};

// block pair p of the upper triangle of MB x MB blocks
template <int MB>
__device__ inline void pair_of(int p, int &bi, int &bj)
{
    bj = 0;
    while ((bj + 1) * (bj + 2) / 2 <= p)
        ++bj;
    bi = p - bj * (bj + 1) / 2;
}

// acc[i] += row block ra of panel a times row block rb + i of panel b over `kbs` contraction blocks; a's fragments serve them all
template <int N>
__device__ inline void multiply_blocks(f32x16 *acc, const Panel &a, int64_t ra, const Panel &b, int64_t rb, int kbs, int lane)
{
#pragma unroll 4
    for (int kb = 0; kb < kbs; ++kb)
    {
        const char *pa = fragment(a, ra, kb, lane);
        const half8 ah = *reinterpret_cast<const half8 *>(pa), al = *reinterpret_cast<const half8 *>(pa + 1024);
        half8 bh[N], bl[N];
#pragma unroll
        for (int i = 0; i < N; ++i)
        {
            const char *pb = fragment(b, rb + i, kb, lane);
            bh[i] = *reinterpret_cast<const half8 *>(pb), bl[i] = *reinterpret_cast<const half8 *>(pb + 1024);
        }
#pragma unroll
        for (int i = 0; i < N; ++i)
            acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bl[i], acc[i], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < N; ++i)
            acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(al, bh[i], acc[i], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < N; ++i)
            acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bh[i], acc[i], 0, 0, 0);
    }
}

// store_mirror through half the scratch, sixteen rows at a time
__device__ inline void store_mirror_halves(const Panel &p, int64_t rb, int64_t cb, int lane, const f32x16 &c, float *scratch)
{
    float v[2][8];
#pragma unroll
    for (int part = 0; part < 2; ++part)
    {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            scratch[(8 * (lane >> 5) + e) * 33 + (lane & 31)] = c[8 * part + e];
        __builtin_amdgcn_wave_barrier();
        if (((lane & 31) >> 4) == part)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    v[h][e] = scratch[(lane & 15) * 33 + 16 * h + 8 * (lane >> 5) + e];
        __builtin_amdgcn_wave_barrier();
    }
    store_fragment(p, rb, cb * 2, lane, v[0]);
    store_fragment(p, rb, cb * 2 + 1, lane, v[1]);
}

__device__ inline void clear(f32x16 &c)
{
#pragma unroll
    for (int e = 0; e < 16; ++e)
        c[e] = 0.f;
}

// MB: blocks of 32 rows (m padded), CB: blocks of 32 columns of a strip
template <int MB, int CB, int MODE>
__global__ __launch_bounds__(MB == 4 ? 512 : 256, 2) void muon_slim_kernel(const SlimArgs s)
{
    constexpr int W = MB == 4 ? 8 : 4, kPairs = MB * (MB + 1) / 2, M = MB * 32, C = CB * 32;
    constexpr int kSquare = MB * MB * 2 * kBlockBytes;                 // an m x m panel
    constexpr int kStrip  = MB * CB * 2 * kBlockBytes;                 // the strip's rows of m
    constexpr int kScratch = W * 32 * 33 * 4, kTileF = M * (C + 1) * 4;
    constexpr int kFirstRegion = kSquare > kScratch ? kSquare : kScratch, kLarger = kSquare > kStrip ? kSquare : kStrip;
    constexpr int kSecond = kLarger > kScratch ? kLarger : kScratch;
    // one strip: X by columns, then what is needed in turn — X by rows, A, b A + c A A —, then half the scratch
    constexpr int kWholeLds = kStrip + (kTileF > kLarger + kScratch / 2 ? kTileF : kLarger + kScratch / 2);
    constexpr int kLds = MODE == kWhole ? kWholeLds : kFirstRegion + kSecond > kTileF + kStrip ? kFirstRegion + kSecond : kTileF + kStrip;
    __shared__ __attribute__((aligned(16))) char lds[kLds];
    __shared__ double norm_parts[W];
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63;
    const int strip = blockIdx.x, z = blockIdx.y;
    const Panel xt{MODE == kWhole ? lds : s.xt + z * s.xt_bytes, MB * 2};
    const int64_t rb0 = (int64_t)strip * CB;  // the strip's first row block in xt
    float *scratch = MODE == kWhole ? reinterpret_cast<float *>(lds + kStrip + kLarger) + wave * (16 * 33) : reinterpret_cast<float *>(lds) + wave * (32 * 33);
    Panel rows{nullptr, CB * 2};  // the strip as rows of m, for its share of A

    if constexpr (MODE == kFirst || MODE == kWhole)
    {
        rows.base  = lds + (MODE == kWhole ? kStrip : kTileF);
        float *tile = reinterpret_cast<float *>(lds + (MODE == kWhole ? kStrip : 0));  // [m][C + 1]
        double factor = 1.0, squares = 0.0;
        if constexpr (MODE == kFirst)
            factor = operand_factor(sum_of_parts<W>(s.sums + (int64_t)z * s.parts, s.parts, norm_parts), s.eps);
        const Update u{s.a.g[z], s.a.buf[z], s.a.momentum, s.a.nesterov};
        const bool tall = s.a.rows > s.a.cols;
        const int64_t m = tall ? s.a.cols : s.a.rows, n = tall ? s.a.rows : s.a.cols, n0 = (int64_t)strip * C;
#pragma unroll 16
        for (int i = threadIdx.x; i < M * C; i += W * 64)
        {
            // lanes along what lies contiguous
            const int r = tall ? i % M : i / C, c = tall ? i / M : i % C;
            float v = 0.f;
            if (r < m && n0 + c < n)
            {
                const int64_t at = tall ? (n0 + c) * m + r : r * n + n0 + c;
                if constexpr (MODE == kWhole)
                {
                    if (u.buf)
                        s.a.buf[z][at] = u.buf[at] * u.momentum + u.g[at];
                    v = u(at);
                    squares += (double)v * (double)v;
                }
                else
                    v = (float)((double)u(at) * factor);
            }
            tile[r * (C + 1) + c] = v;
        }
        if constexpr (MODE == kWhole)
        {
#pragma unroll
            for (int o = 32; o > 0; o >>= 1)
                squares += __shfl_xor(squares, o, 64);
            if (lane == 0)
                norm_parts[wave] = squares;
            __syncthreads();
            squares = norm_parts[0];
#pragma unroll
            for (int w = 1; w < W; ++w)
                squares += norm_parts[w];
            factor = operand_factor(squares, s.eps);
        }
        else
        {
            __syncthreads();
            factor = 1.0;  // applied already
        }
        for (int f = wave; f < CB * MB * 2; f += W)
        {
            const int cb = f / (MB * 2), kb = f % (MB * 2);
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
                v[e] = (float)((double)tile[(kb * 16 + (lane >> 5) * 8 + e) * (C + 1) + cb * 32 + (lane & 31)] * factor);
            store_fragment(xt, rb0 + cb, kb, lane, v);
        }
        float v[MB * CB * 2 / W][8];
#pragma unroll
        for (int i = 0; i < MB * CB * 2 / W; ++i)
        {
            const int f = wave + i * W, rb = f / (CB * 2), kb = f % (CB * 2);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                v[i][e] = (float)((double)tile[(rb * 32 + (lane & 31)) * (C + 1) + kb * 16 + (lane >> 5) * 8 + e] * factor);
        }
        if constexpr (MODE == kWhole)
            __syncthreads();  // the rows go where the values came from
#pragma unroll
        for (int i = 0; i < MB * CB * 2 / W; ++i)
        {
            const int f = wave + i * W, rb = f / (CB * 2), kb = f % (CB * 2);
            store_fragment(rows, rb, kb, lane, v[i]);
        }
    }
    constexpr int PP = (kPairs + W - 1) / W;
    constexpr int kSquareBlocks = MB * MB / W, kStripBlocks = MB * CB / W;  // a wave's: one row block of m, neighbouring columns
    const Panel square{lds + (MODE == kWhole ? kStrip : 0), MB * 2}, poly{lds + (MODE == kWhole ? kStrip : kFirstRegion), MB * 2};
    if constexpr (MODE == kWhole)
        __syncthreads();
    for (int k = 1;; ++k)
    {
        if constexpr (MODE != kFirst)
        {
            if constexpr (MODE == kWhole)
            {
                // A of the one strip there is: every block
                f32x16 a[kSquareBlocks];
                for (f32x16 &c : a)
                    clear(c);
                multiply_blocks<kSquareBlocks>(a, rows, wave % MB, rows, wave / MB * kSquareBlocks, CB * 2, lane);
                __syncthreads();  // A goes where the rows lie
#pragma unroll
                for (int i = 0; i < kSquareBlocks; ++i)
                {
                    to_columns(a[i]);
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        a[i][e] *= 1.f / kScale;
                    store_columns(square, wave / MB * kSquareBlocks + i, wave % MB, lane, a[i]);
                }
            }
            else
            {
                // A from the strips' shares of its upper triangle, in strip order
#pragma unroll
                for (int i = 0; i < PP; ++i)
                {
                    const int p = wave + i * W;
                    if (p >= kPairs)
                        continue;
                    f32x16 a;
                    clear(a);
                    const f32x4 *in = s.share_in + ((int64_t)z * s.strips * kPairs + p) * 256 + lane;
#pragma unroll 8
                    for (int t = 0; t < s.strips; ++t)
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                        {
                            const f32x4 v = in[(int64_t)t * kPairs * 256 + q * 64];
                            a[4 * q] += v[0], a[4 * q + 1] += v[1], a[4 * q + 2] += v[2], a[4 * q + 3] += v[3];
                        }
                    to_columns(a);
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        a[e] *= 1.f / kScale;
                    int bi, bj;
                    pair_of<MB>(p, bi, bj);
                    store_columns(square, bj, bi, lane, a);
                    // the mirrored block: lane's row and column change places through the other region
                    if (bi != bj)
                        store_mirror(square, bi, bj, lane, a, reinterpret_cast<float *>(lds + kFirstRegion) + wave * (32 * 33));
                }
            }
            __syncthreads();
            f32x16 b[kSquareBlocks];
            for (f32x16 &c : b)
                clear(c);
            multiply_blocks<kSquareBlocks>(b, square, wave % MB, square, wave / MB * kSquareBlocks, MB * 2, lane);
#pragma unroll
            for (int i = 0; i < kSquareBlocks; ++i)
            {
                const int bj = wave / MB * kSquareBlocks + i;
                to_columns(b[i]);
                combine(b[i], square, bj, wave % MB, lane, s.cc / kScale, s.cb);
            }
            if constexpr (MODE == kWhole)
                __syncthreads();  // b A + c A A goes where A lies
#pragma unroll
            for (int i = 0; i < kSquareBlocks; ++i)
                store_columns(poly, wave / MB * kSquareBlocks + i, wave % MB, lane, b[i]);
            __syncthreads();
            const bool last = MODE == kLast || (MODE == kWhole && k == s.steps);
            const int rb = wave % MB, cb0 = wave / MB * kStripBlocks;
            f32x16 x[kStripBlocks];
            for (f32x16 &c : x)
                clear(c);
            multiply_blocks<kStripBlocks>(x, poly, rb, xt, rb0 + cb0, MB * 2, lane);
#pragma unroll
            for (int i = 0; i < kStripBlocks; ++i)
            {
                to_columns(x[i]);
                combine(x[i], xt, rb0 + cb0 + i, rb, lane, 1.f / kScale, s.ca);
            }
            if (last)
            {
#pragma unroll
                for (int i = 0; i < kStripBlocks; ++i)
                {
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        x[i][e] *= 1.f / kScale;
                    write_result(s.a, z, x[i], rb, rb0 + cb0 + i, lane, s.keep);
                }
                return;
            }
            __syncthreads();  // every wave has read its blocks of X and of b A + c A A
            rows.base = lds + (MODE == kWhole ? kStrip : kFirstRegion);
#pragma unroll
            for (int i = 0; i < kStripBlocks; ++i)
            {
                store_columns(xt, rb0 + cb0 + i, rb, lane, x[i]);
                if constexpr (MODE == kWhole)
                    store_mirror_halves(rows, rb, cb0 + i, lane, x[i], scratch);
                else
                    store_mirror(rows, rb, cb0 + i, lane, x[i], scratch);
            }
        }
        __syncthreads();
        if constexpr (MODE != kWhole)
            break;
    }
    for (int p = wave; p < kPairs; p += W)
    {
        int bi, bj;
        pair_of<MB>(p, bi, bj);
        f32x16 c;
        clear(c);
        multiply_blocks<1>(&c, rows, bi, rows, bj, CB * 2, lane);
        f32x4 *out = s.share_out + (((int64_t)z * s.strips + strip) * kPairs + p) * 256 + lane;
#pragma unroll
        for (int q = 0; q < 4; ++q)
            out[q * 64] = f32x4{c[4 * q], c[4 * q + 1], c[4 * q + 2], c[4 * q + 3]};
    }
}

struct Shape
{
    int64_t m, n;
    int mb, cb, strips;
    int64_t xt_bytes, share_bytes;
};

Shape shape_of(int64_t rows, int64_t cols)
{
    Shape s;
    s.m = std::min(rows, cols), s.n = std::max(rows, cols);
    s.mb = s.m <= 64 ? 2 : 4, s.cb = s.n <= 64 || (s.n > 128 && s.n <= 512) ? 2 : 4;
    s.strips      = (int)odl::ceil_div(s.n, s.cb * 32);
    s.xt_bytes    = (int64_t)s.strips * s.cb * s.mb * 2 * kBlockBytes;
    s.share_bytes = (int64_t)s.strips * (s.mb * (s.mb + 1) / 2) * 4096;
    return s;
}

template <int MB, int CB>
void launch(int mode, dim3 grid, const SlimArgs &a, hipStream_t st)
{
    const dim3 block(MB == 4 ? 512 : 256);
    if (mode == kFirst)
        muon_slim_kernel<MB, CB, kFirst><<<grid, block, 0, st>>>(a);
    else if (mode == kStep)
        muon_slim_kernel<MB, CB, kStep><<<grid, block, 0, st>>>(a);
    else if (mode == kLast)
        muon_slim_kernel<MB, CB, kLast><<<grid, block, 0, st>>>(a);
    else if constexpr (MB <= CB)  // m <= n
        muon_slim_kernel<MB, CB, kWhole><<<grid, block, 0, st>>>(a);
}
}  // namespace

namespace odl
{
namespace muon
{
bool slim_fits(int64_t rows, int64_t cols)
{
    return std::min(rows, cols) <= kMostM && std::max(rows, cols) <= kMostN;
}

bool slim_whole(int64_t rows, int64_t cols)
{
    return std::max(rows, cols) <= kMostM;
}

size_t slim_bytes(int64_t rows, int64_t cols)
{
    const Shape s = shape_of(rows, cols);
    return (size_t)(s.xt_bytes + 2 * s.share_bytes);
}

int slim_run(const Matrices &mat, int count, const Settings &set, const double *sums, int parts, char *workspace, hipStream_t st)
{
    const Shape sh = shape_of(mat.rows, mat.cols);
    SlimArgs s{};
    s.a = mat, s.sums = sums, s.parts = parts, s.steps = set.steps, s.eps = (double)set.eps;
    s.xt = workspace, s.xt_bytes = sh.xt_bytes, s.strips = sh.strips;
    s.ca = set.a, s.cb = set.b, s.cc = set.c, s.keep = set.keep;
    char *shares[2] = {workspace + count * sh.xt_bytes, workspace + count * (sh.xt_bytes + sh.share_bytes)};
    const dim3 grid((unsigned)sh.strips, (unsigned)count);
    const bool whole = slim_whole(mat.rows, mat.cols);
    for (int k = 0; k <= (whole ? 0 : set.steps); ++k)
    {
        s.share_in  = reinterpret_cast<const f32x4 *>(shares[(k + 1) & 1]);
        s.share_out = reinterpret_cast<f32x4 *>(shares[k & 1]);
        const int mode = whole ? kWhole : k == 0 ? kFirst : k == set.steps ? kLast : kStep;
        if (sh.mb == 2 && sh.cb == 2)
            launch<2, 2>(mode, grid, s, st);
        else if (sh.mb == 2)
            launch<2, 4>(mode, grid, s, st);
        else if (sh.cb == 2)
            launch<4, 2>(mode, grid, s, st);
        else
            launch<4, 4>(mode, grid, s, st);
        ODL_LAUNCH_CHECK();
    }
    return ODL_OK;
}
}  // namespace muon
}  // namespace odl
