// Orthogonalised updates: Newton-Schulz steps on a matrix (or a list of equal ones), and the optimiser step around them.
//
//   X0 = U / (||U||_F + eps), transposed if it has more rows than columns (m <= n from here on)
//   X <- a X + (b A + c A A) X,  A = X X^T        `steps` times
//   U: the gradient; in the optimiser step the momentum buf <- mu buf + g, or g + mu buf (Nesterov)
//   p <- p (1 - lr * weight_decay) - lr * sqrt(max(1, outputs / inputs)) * X       [outputs, inputs] or [inputs, outputs]
//
// What bounds it: three products a step, 2m^2 n + 2m^3 + 2m^2 n operations, of which the two symmetric ones need only half of
// their tiles. They run as three float16 products each (split_gemm.h); X, A and b A + c A A live only as operands of
// those, between launches in L2 and the memory-side cache. Every epilogue writes its result as the next product's operands: X
// as rows of m (for X X^T) and as rows of n (for B X), the symmetric ones with their mirror image. The last one writes X, or
// applies it to the parameter.
//
// Measured: 4096 x 4096, five steps: 4.0 to 4.15 ms, 331 to 343 TFLOP/s of the work that symmetry leaves (the chip's power limit
// for these products is 425 to 455); 1000 x 1000: 172 us, seventeen launches of which each waits for the one before (a product of
// these sizes takes 10 to 12 us, its operations alone 3).
//
// Singular values of X stay under max |f| on [0, 1], f(s) = a s + b s^3 + c s^5 (1.21 for the usual coefficients), so all
// operands are scaled by the same 2^13: float16 holds 8 * 2^13, and coefficients that lead A = X X^T (the singular values'
// squares) or b A + c A A past 7.5 are refused.
#include <cmath>

#include "muon.h"

namespace
{
using namespace odl::split;
using namespace odl::muon;

// buf <- mu buf + g, and the partial sums of U's squares, in 64 bits: the norm's error is common to all of X, and the steps
// amplify it
__global__ __launch_bounds__(kBlock) void muon_norm_kernel(const Matrices a, double *sums)
{
    __shared__ double part[4];
    const int z = blockIdx.y;
    const int64_t n = a.rows * a.cols;
    float *buf = a.buf[z];
    const Update u{a.g[z], buf, a.momentum, a.nesterov};
    double s = 0.0;
    const int64_t step = (int64_t)gridDim.x * kBlock, at = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    // four at a time where the rows of 16 bytes allow it; the rest one by one
    const int64_t quads = ((reinterpret_cast<uintptr_t>(u.g) | reinterpret_cast<uintptr_t>(buf)) & 15) == 0 ? n / 4 : 0;
    for (int64_t i = at; i < quads; i += step)
    {
        f32x4 g = reinterpret_cast<const f32x4 *>(u.g)[i];
        if (buf)
        {
            f32x4 m = reinterpret_cast<f32x4 *>(buf)[i];
            m = m * a.momentum + g;
            reinterpret_cast<f32x4 *>(buf)[i] = m;
            g = a.nesterov ? g + a.momentum * m : m;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            s += (double)g[e] * (double)g[e];
    }
    for (int64_t i = quads * 4 + at; i < n; i += step)
    {
        if (buf)
            buf[i] = buf[i] * a.momentum + u.g[i];
        const double v = (double)u(i);
        s += v * v;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0)
        part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0)
        sums[(int64_t)z * gridDim.x + blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
}

// X0 as panels: r has the matrix's rows as rows, t its columns
__global__ __launch_bounds__(kBlock) void muon_prepare_kernel(const Matrices a, const double *sums, int parts, double eps, Panel r, Panel t,
                                                              int64_t batch_bytes)
{
    __shared__ float tile[64][65];
    __shared__ double part[4];
    const int z = blockIdx.z;
    r.base += z * batch_bytes, t.base += z * batch_bytes;
    const auto factor = [&] { return operand_factor(sum_of_parts<4>(sums + (int64_t)z * parts, parts, part), eps); };
    split_tile(UpdateAt{{a.g[z], a.buf[z], a.momentum, a.nesterov}, a.cols}, factor, a.rows, a.cols, (int64_t)blockIdx.y * 64, (int64_t)blockIdx.x * 64, r, t, tile);
}

// A = X X^T (prev null), or b A + c A A: symmetric, computed for tile row <= tile column
struct SymmetricEpilogue
{
    Panel out, prev;
    int64_t batch_bytes;
    float own, before;
    template <class T, class Acc>
    __device__ void operator()(const T &t, Acc &acc) const
    {
        Panel o = out, q = prev;
        o.base += t.z * batch_bytes;
        if (q.base)
            q.base += t.z * batch_bytes;
#pragma unroll
        for (int mi = 0; mi < T::MI; ++mi)
#pragma unroll
            for (int ni = 0; ni < T::NI; ++ni)
            {
                f32x16 &c = acc[mi][ni];
                const int64_t rb = t.row_block(mi), cb = t.col_block(ni);
                to_columns(c);
                if (q.base)
                    combine(c, q, cb, rb, t.lane, own, before);
                else
                {
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        c[e] *= own;
                }
                store_columns(o, cb, rb, t.lane, c);
                if (t.tm != t.tn)
                    store_mirror(o, rb, cb, t.lane, c, t.wave_scratch());
            }
    }
};

// X <- a X + B X, as rows of n (columns of this product) and rows of m
struct StepEpilogue
{
    Panel prev, columns, rows;
    int64_t batch_bytes;
    float own, before;
    template <class T, class Acc>
    __device__ void operator()(const T &t, Acc &acc) const
    {
        Panel q = prev, oc = columns, orow = rows;
        q.base += t.z * batch_bytes, oc.base += t.z * batch_bytes, orow.base += t.z * batch_bytes;
#pragma unroll
        for (int mi = 0; mi < T::MI; ++mi)
#pragma unroll
            for (int ni = 0; ni < T::NI; ++ni)
            {
                f32x16 &c = acc[mi][ni];
                const int64_t rb = t.row_block(mi), cb = t.col_block(ni);
                to_columns(c);
                combine(c, q, cb, rb, t.lane, own, before);
                store_columns(oc, cb, rb, t.lane, c);
                store_mirror(orow, rb, cb, t.lane, c, t.wave_scratch());
            }
    }
};

// the last step: X itself, or the parameter it updates
struct LastEpilogue
{
    Panel prev;
    int64_t batch_bytes;
    float own, before;
    Matrices a;
    float keep;  // p * keep - X * rate
    template <class T, class Acc>
    __device__ void operator()(const T &t, Acc &acc) const
    {
        Panel q = prev;
        q.base += t.z * batch_bytes;
#pragma unroll
        for (int mi = 0; mi < T::MI; ++mi)
#pragma unroll
            for (int ni = 0; ni < T::NI; ++ni)
            {
                f32x16 &c = acc[mi][ni];
                const int64_t rb = t.row_block(mi), cb = t.col_block(ni);
                to_columns(c);
                combine(c, q, cb, rb, t.lane, own, before);
                write_result(a, t.z, c, rb, cb, t.lane, keep);
            }
    }
};

struct Space
{
    double *sums;
    Panel xr[2], xt[2], a, b;
    int64_t batch_bytes;
    Cut gram, poly, step;
    void *parts;  // of a product whose contraction is cut
    size_t bytes;
};

int norm_blocks(int64_t elements)
{
    return (int)std::min<int64_t>(1024, std::max<int64_t>(1, odl::ceil_div(elements, 2048)));
}

Space space_for(char *base, int count, int64_t rows, int64_t cols)
{
    const int64_t mp = padded(std::min(rows, cols)), np = padded(std::max(rows, cols));
    Space s;
    const int64_t sums = (odl::ceil_div((int64_t)count * norm_blocks(rows * cols) * 8, 256)) * 256;
    const int64_t xb = panel_bytes(mp, np), ab = panel_bytes(mp, mp);
    s.batch_bytes = slim_fits(rows, cols) ? (int64_t)slim_bytes(rows, cols) : 4 * xb + 2 * ab;
    char *at      = base + sums;
    s.sums        = reinterpret_cast<double *>(base);
    for (int i = 0; i < 2; ++i)
        s.xr[i] = Panel{at + 2 * i * xb, np / 16}, s.xt[i] = Panel{at + (2 * i + 1) * xb, mp / 16};
    s.a     = Panel{at + 4 * xb, mp / 16};
    s.b     = Panel{at + 4 * xb + ab, mp / 16};
    s.bytes = (size_t)(sums + count * s.batch_bytes);
    s.parts = base + s.bytes;
    if (!slim_fits(rows, cols))
    {
        const int kb_m = contraction_blocks(std::min(rows, cols)), kb_n = contraction_blocks(std::max(rows, cols));
        const double square = 2.0 * (double)count * mp * (mp + 64), whole = 4.0 * (double)count * mp * np;
        // a step passes on what its sums round, up to 3.4 times: long ones are kept apart (4096 x 4096, against 64 bits: 6.5e-6
        // with one set of accumulators, 3.0e-6 for float32 products in quarters)
        const bool exact = kb_m > 64;
        s.gram = pick_cut(mp, mp, true, count, kb_n, true, square, exact), s.poly = pick_cut(mp, mp, true, count, kb_m, true, square, exact);
        s.step = pick_cut(mp, np, false, count, kb_m, true, whole, exact);
        s.bytes += std::max({part_bytes(s.gram, mp, mp, count), part_bytes(s.poly, mp, mp, count), part_bytes(s.step, mp, np, count)});
    }
    return s;
}

// how many equal matrices go through the launches together: what 2 GiB of workspace holds. The last group of a call may be
// smaller, and its products cut into more runs than the full group's: either may need the larger workspace.
int group_of(int count, int64_t rows, int64_t cols)
{
    const int64_t each = space_for(nullptr, 1, rows, cols).batch_bytes;
    return (int)std::max<int64_t>(1, std::min<int64_t>(std::min(count, kGroup), ((int64_t)2 << 30) / each));
}

// Where f's iterates take singular values from [0, 1], and what b t + c t^2 (t = s^2) reaches on the way.
bool coefficients_ok(double a, double b, double c, int steps)
{
    double top = 1.0;
    for (int k = 0; k < steps; ++k)
    {
        double next = 0.0;
        for (int i = 0; i <= 2048; ++i)
        {
            const double s = top * i / 2048, t = s * s, poly = b * t + c * t * t;
            const double f = std::fabs(s * (a + poly));
            if (!(f * f < kMost && std::fabs(poly) < kMost))  // (false for NaN too)
                return false;
            next = std::max(next, f);
        }
        // f may also lift what rounding left under the last top
        top = std::max(next, 1.0);
    }
    return true;
}

constexpr int64_t kMostSide = (int64_t)1 << 20;

int check_common(const char *who, int64_t rows, int64_t cols, int steps, float a, float b, float c, float eps)
{
    ODL_REQUIRE(rows >= 0 && cols >= 0 && rows <= kMostSide && cols <= kMostSide, "%s: sides of 0 to %lld, got [%lld, %lld]", who, (long long)kMostSide,
                (long long)rows, (long long)cols);
    ODL_REQUIRE(steps >= 1 && steps <= 100, "%s: 1 to 100 steps, got %d", who, steps);
    ODL_REQUIRE(eps >= 0.f, "%s: eps must not be negative, got %g", who, (double)eps);
    ODL_REQUIRE(coefficients_ok(a, b, c, steps), "%s: coefficients (%g, %g, %g) take singular values past the range of the products' operands", who, (double)a,
                (double)b, (double)c);
    return ODL_OK;
}

int run_group(const char *who, const Matrices &mat, int count, int steps, float a, float b, float c, float eps, float keep, void *workspace,
              size_t workspace_bytes, hipStream_t st)
{
    const Space s = space_for(static_cast<char *>(workspace), count, mat.rows, mat.cols);
    ODL_REQUIRE(s.bytes <= workspace_bytes, "%s: workspace of %zu bytes needed for %d of [%lld, %lld], got %zu", who, s.bytes, count, (long long)mat.rows,
                (long long)mat.cols, workspace_bytes);
    const bool tall  = mat.rows > mat.cols;
    const int64_t m = std::min(mat.rows, mat.cols), n = std::max(mat.rows, mat.cols), mp = padded(m), np = padded(n);
    const int parts = norm_blocks(mat.rows * mat.cols);
    if (!slim_whole(mat.rows, mat.cols))
    {
        muon_norm_kernel<<<dim3((unsigned)parts, (unsigned)count), dim3(kBlock), 0, st>>>(mat, s.sums);
        ODL_LAUNCH_CHECK();
    }
    if (slim_fits(mat.rows, mat.cols))
        return slim_run(mat, count, Settings{steps, a, b, c, eps, keep}, s.sums, parts, s.xr[0].base, st);
    const int64_t rp = tall ? np : mp, cp = tall ? mp : np;
    muon_prepare_kernel<<<dim3((unsigned)(cp / 64), (unsigned)(rp / 64), (unsigned)count), dim3(kBlock), 0, st>>>(
        mat, s.sums, parts, (double)eps, tall ? s.xt[0] : s.xr[0], tall ? s.xr[0] : s.xt[0], s.batch_bytes);
    ODL_LAUNCH_CHECK();
    const int kb_m = contraction_blocks(m), kb_n = contraction_blocks(n);
    for (int k = 0; k < steps; ++k)
    {
        const Panel xr = s.xr[k & 1], xt = s.xt[k & 1];
        GemmArgs g{};
        g.batch = count, g.a_batch = g.b_batch = s.batch_bytes;
        g.symmetric = 1;
        g.a = xr, g.b = xr, g.nkb = kb_n;
        if (int rc = launch_whole_gemm(g, mp, mp, s.gram, s.parts, SymmetricEpilogue{s.a, Panel{nullptr, 0}, s.batch_bytes, 1.f / kScale, 0.f}, st))
            return rc;
        g.a = s.a, g.b = s.a, g.nkb = kb_m;
        if (int rc = launch_whole_gemm(g, mp, mp, s.poly, s.parts, SymmetricEpilogue{s.b, s.a, s.batch_bytes, c / kScale, b}, st))
            return rc;
        g.symmetric = 0;
        g.a = s.b, g.b = xt;
        int rc;
        if (k + 1 < steps)
            rc = launch_whole_gemm(g, mp, np, s.step, s.parts, StepEpilogue{xt, s.xt[(k + 1) & 1], s.xr[(k + 1) & 1], s.batch_bytes, 1.f / kScale, a}, st);
        else
            rc = launch_whole_gemm(g, mp, np, s.step, s.parts, LastEpilogue{xt, s.batch_bytes, 1.f / kScale / kScale, a / kScale, mat, keep}, st);
        if (rc)
            return rc;
    }
    return ODL_OK;
}
}  // namespace

extern "C" size_t odl_hip_newton_schulz_workspace_bytes(int64_t batch, int64_t rows, int64_t cols)
{
    if (batch <= 0 || rows <= 0 || cols <= 0 || rows > kMostSide || cols > kMostSide)
        return 0;
    const int group = group_of((int)std::min<int64_t>(batch, kGroup), rows, cols), rest = (int)(batch % group);
    return std::max(space_for(nullptr, group, rows, cols).bytes, rest ? space_for(nullptr, rest, rows, cols).bytes : (size_t)0);
}

extern "C" int odl_hip_newton_schulz(const float *g, int64_t batch, int64_t rows, int64_t cols, int steps, float a, float b, float c, float eps, float *out,
                                     void *workspace, size_t workspace_bytes, void *stream)
{
    const char *who = "newton_schulz";
    ODL_REQUIRE(batch >= 0, "%s: negative batch", who);
    if (int rc = check_common(who, rows, cols, steps, a, b, c, eps))
        return rc;
    if (batch == 0 || rows == 0 || cols == 0)
        return ODL_OK;
    ODL_REQUIRE(g && out, "%s: null argument", who);
    const size_t need = odl_hip_newton_schulz_workspace_bytes(batch, rows, cols);
    ODL_REQUIRE(workspace && workspace_bytes >= need, "%s: workspace of %zu bytes needed, got %zu", who, need, workspace ? workspace_bytes : (size_t)0);
    ODL_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "%s: the workspace must be 16-byte aligned", who);
    ODL_REQUIRE_DEVICE();
    const int group = group_of((int)std::min<int64_t>(batch, kGroup), rows, cols);
    for (int64_t first = 0; first < batch; first += group)
    {
        const int count = (int)std::min<int64_t>(group, batch - first);
        Matrices mat{};
        mat.rows = rows, mat.cols = cols;
        for (int i = 0; i < count; ++i)
            mat.g[i] = g + (first + i) * rows * cols, mat.out[i] = out + (first + i) * rows * cols;
        if (int rc = run_group(who, mat, count, steps, a, b, c, eps, 1.f, workspace, workspace_bytes, odl::as_stream(stream)))
            return rc;
    }
    return ODL_OK;
}

extern "C" size_t odl_hip_muon_step_multi_workspace_bytes(int count, const int64_t *host_rows, const int64_t *host_cols)
{
    size_t most = 0;
    for (int i = 0; i < count && host_rows && host_cols; ++i)
    {
        int equal = 0;
        for (int j = 0; j < count; ++j)
            equal += host_rows[j] == host_rows[i] && host_cols[j] == host_cols[i];
        most = std::max(most, odl_hip_newton_schulz_workspace_bytes(equal, host_rows[i], host_cols[i]));
    }
    return most;
}

extern "C" int odl_hip_muon_step_multi(int count, const float *const *p, const float *const *g, float *const *buf, const int64_t *host_rows,
                                       const int64_t *host_cols, float lr, float momentum, int nesterov, float weight_decay, int steps, float a, float b,
                                       float c, float eps, float *const *p_out, void *workspace, size_t workspace_bytes, void *stream)
{
    return odl_hip_muon_step_multi_in_out(count, p, g, buf, host_rows, host_cols, nullptr, lr, momentum, nesterov, weight_decay, steps, a, b, c, eps, p_out,
                                          workspace, workspace_bytes, stream);
}

extern "C" int odl_hip_muon_step_multi_in_out(int count, const float *const *p, const float *const *g, float *const *buf, const int64_t *host_rows,
                                              const int64_t *host_cols, const int *host_in_out, float lr, float momentum, int nesterov, float weight_decay,
                                              int steps, float a, float b, float c, float eps, float *const *p_out, void *workspace,
                                              size_t workspace_bytes, void *stream)
{
    const char *who = "muon_step_multi";
    ODL_REQUIRE(count >= 0, "%s: negative count", who);
    if (count == 0)
        return ODL_OK;
    ODL_REQUIRE(p && g && buf && host_rows && host_cols && p_out, "%s: null argument", who);
    for (int i = 0; i < count; ++i)
    {
        if (int rc = check_common(who, host_rows[i], host_cols[i], i == 0 ? steps : 1, i == 0 ? a : 1.f, i == 0 ? b : 0.f, i == 0 ? c : 0.f, eps))
            return rc;
        if (host_rows[i] * host_cols[i] == 0)
            continue;
        ODL_REQUIRE(p[i] && g[i] && buf[i] && p_out[i], "%s: null pointer for entry %d", who, i);
        for (int j = 0; j < i; ++j)
            ODL_REQUIRE(host_rows[j] * host_cols[j] == 0 || (buf[j] != buf[i] && p_out[j] != p_out[i]),
                        "%s: entries %d and %d write the same momentum or parameter", who, j, i);
    }
    const size_t need = odl_hip_muon_step_multi_workspace_bytes(count, host_rows, host_cols);
    ODL_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "%s: workspace of %zu bytes needed, got %zu", who, need,
                workspace ? workspace_bytes : (size_t)0);
    ODL_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "%s: the workspace must be 16-byte aligned", who);
    ODL_REQUIRE_DEVICE();
    for (int i = 0; i < count; ++i)
    {
        const int64_t rows = host_rows[i], cols = host_cols[i];
        bool done = rows == 0 || cols == 0;
        for (int j = 0; j < i && !done; ++j)
            done = host_rows[j] == rows && host_cols[j] == cols;
        if (done)
            continue;
        // all entries of this shape, a group at a time
        int equal = 0;
        for (int j = i; j < count; ++j)
            equal += host_rows[j] == rows && host_cols[j] == cols;
        const int group = group_of(std::min(equal, kGroup), rows, cols);
        Matrices mat{};
        mat.rows = rows, mat.cols = cols, mat.momentum = momentum, mat.nesterov = nesterov;
        int in = 0;
        for (int j = i; j < count; ++j)
        {
            if (host_rows[j] != rows || host_cols[j] != cols)
                continue;
            mat.g[in] = g[j], mat.buf[in] = buf[j], mat.p[in] = p[j], mat.out[in] = p_out[j];
            const bool in_out = host_in_out && host_in_out[j];
            mat.rate[in] = lr * (float)std::sqrt(std::max(1.0, in_out ? (double)cols / (double)rows : (double)rows / (double)cols));
            ++in, --equal;
            if (in == group || equal == 0)
            {
                if (int rc = run_group(who, mat, in, steps, a, b, c, eps, 1.f - lr * weight_decay, workspace, workspace_bytes, odl::as_stream(stream)))
                    return rc;
                in = 0;
            }
        }
    }
    return ODL_OK;
}
