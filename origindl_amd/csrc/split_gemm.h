// Float32 products on the float16 matrix instructions of gfx950, for the operators whose products are large and whose
// epilogues do the rest of the operator's work (linear_ce.hip, muon.hip).
//
// Mathematics. A float32 operand, scaled by a power of two that brings its largest magnitude to [2^14, 2^15), is the sum of
// two float16 numbers and an error: hi = fp16(x), lo = fp16(x - hi), |x - hi - lo| <= 2^-22 |x| (elements under 2^-17 of the
// largest: 2^-25, half the spacing of float16's smallest numbers, which is 2^-39 of a largest one of 2^14). Then
//     a . b = ah.bh + ah.bl + al.bh     (+ al.bl <= 2^-22 |a||b|, left out)
// with every product exact in float32 and all three summed in float32: the error of a float32 product's own sums (operators
// against 64 bits: 0.1 to 1.0 times that of the float32 library's products, 1.3 times over five steps of 4096-wide symmetric
// products), at three float16 matrix instructions instead of the sixteen times slower float32 one.
//
// Layout ("panel"). An operand [rows, contraction] lies as blocks of 32 rows x 16 contraction values, 2 KB each: 1 KB of hi,
// then 1 KB of lo, each in the order in which v_mfma_f32_32x32x16_f16 takes it (lane l: row l % 32, contraction values
// 8 * (l / 32) .. + 7). Blocks of a row block are consecutive along the contraction. A load into LDS is then a straight copy
// of 16 bytes a lane, a fragment is one ds_read_b128 without bank conflicts, and rows, columns and contraction values past
// the matrix are zeros in memory, so the product's loop has no edges.
//
// Sums. Every product added to an accumulator rounds it once more, the small cross terms too. Where registers allow (all tiles
// but 256 x 256) the cross terms have accumulators of their own, which join the others at the end: a third of the roundings.
//
// The product. A workgroup holds a BM x BN tile; four stages of one contraction block each travel into LDS by direct loads
// (no registers), queued four stages ahead; fragments of the next block are read while the present block multiplies. A
// stage's three products use 4 fragments a pair of blocks where a plain float16 product reads 2 for one: two thirds of the LDS
// reads per matrix instruction. What bounds it is the chip's power: 425 to 456 TFLOP/s of float32 products, 1.3 PFLOP/s of
// matrix instructions, whichever large tile is taken (the library's float16 product: 1.1 to 1.2; its float32 product: 0.15).
#pragma once
#include <algorithm>
#include <type_traits>

#include "odl_common.h"

namespace odl
{
namespace split
{
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int kBlockBytes = 2048;  // 32 rows x 16 contraction values, hi and lo
constexpr int kStages     = 4;

// A panel: where it lies and how many blocks a row block holds.
struct Panel
{
    char *base;
    int64_t kb;  // contraction blocks allocated per row block

    __host__ __device__ int64_t row_block_bytes() const { return kb * kBlockBytes; }
};

// contraction blocks of a product
inline int contraction_blocks(int64_t contraction)
{
    return (int)ceil_div(contraction, 32) * 2;
}

inline int64_t panel_bytes(int64_t rows_pad, int64_t contraction_pad)
{
    return rows_pad * contraction_pad * 4;
}

// Padded extent of a dimension that tiles will cover.
inline int64_t padded(int64_t n)
{
    const int64_t t = n > 64 ? 128 : 64;
    return ceil_div(n, t) * t;
}

// Two values into hi and lo, both rounded to nearest. The mixed-precision multiply-add takes a float16 as it lies in half a
// register: x - hi is one instruction, where converting hi back first would take two.
typedef _Float16 half2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
__device__ inline void split_pair(float x, float y, unsigned &hi, unsigned &lo)
{
    hi = __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2){x, y}, half2));
    float rx, ry;
    asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel_hi:[1,0,0]" : "=v"(rx) : "v"(hi), "v"(x));
    asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(ry) : "v"(hi), "v"(y));
    lo = __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2){rx, ry}, half2));
}
// hi + lo
__device__ inline void join_pair(unsigned hi, unsigned lo, float &x, float &y)
{
    asm("v_fma_mix_f32 %0, %1, 1.0, %2 op_sel_hi:[1,0,1]" : "=v"(x) : "v"(hi), "v"(lo));
    asm("v_fma_mix_f32 %0, %1, 1.0, %2 op_sel:[1,0,1] op_sel_hi:[1,0,1]" : "=v"(y) : "v"(hi), "v"(lo));
}

// where lane `lane` keeps its 8 values (hi; lo follows 1024 bytes later) of block (row block rb, contraction block kb)
__device__ inline char *fragment(const Panel &p, int64_t rb, int64_t kb, int lane)
{
    return p.base + (rb * p.kb + kb) * kBlockBytes + lane * 16;
}

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
__device__ inline void store_fragment(const Panel &p, int64_t rb, int64_t kb, int lane, const float *v)
{
    u32x4 hi, lo;
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        unsigned h, l;
        split_pair(v[2 * i], v[2 * i + 1], h, l);
        hi[i] = h, lo[i] = l;
    }
    char *at = fragment(p, rb, kb, lane);
    *reinterpret_cast<u32x4 *>(at)        = hi;
    *reinterpret_cast<u32x4 *>(at + 1024) = lo;
}

__device__ inline void load_fragment(const Panel &p, int64_t rb, int64_t kb, int lane, float *v)
{
    const char *at = fragment(p, rb, kb, lane);
    const u32x4 hi = *reinterpret_cast<const u32x4 *>(at), lo = *reinterpret_cast<const u32x4 *>(at + 1024);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        join_pair(hi[i], lo[i], v[2 * i], v[2 * i + 1]);
}

// 16 bytes a lane from a buffer into LDS: lane i's data lands at lds_byte_address + 16 * i. An instruction and not the
// compiler's builtin, which would wait for all queued loads before every LDS read; the waits are placed by hand. (One wait
// state between the write of m0 and the load that reads it: inside the asm the compiler does not add it.)
__device__ inline void load_to_lds_16(i32x4 rsrc, unsigned lds_byte_address, unsigned lane_offset, unsigned offset)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 :
                 : "s"(lds_byte_address), "v"(lane_offset), "s"(rsrc), "s"(offset)
                 : "memory", "m0");
}

__device__ inline i32x4 buffer_of(const char *base)
{
    const uint64_t p = reinterpret_cast<uint64_t>(base);
    i32x4 r;
    r[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)p);
    r[1] = __builtin_amdgcn_readfirstlane((int)(uint32_t)(p >> 32));  // stride 0: a raw buffer
    r[2] = 0x7fffffff;
    r[3] = 0x00020000;
    return r;
}

// waits until at most `vm` of the wave's vector-memory operations are outstanding and all of its LDS reads are done
template <int vm>
__device__ inline void wait_loads_and_lds()
{
    static_assert(vm >= 0 && vm < 64, "vmcnt is a 6-bit counter");
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(vm) : "memory");
}
__device__ inline void barrier()
{
    asm volatile("s_barrier" ::: "memory");
}

// A 32x32 accumulator block holds, in lane l, column l % 32 and rows 8q + 4(l / 32) + r in element 4q + r. Exchanging halves of
// the wave between neighbouring quads leaves rows 8(l / 32) + e in element e and 16 + 8(l / 32) + e in element 8 + e: eight
// consecutive rows of one column, which is a lane's part of a fragment of the transposed block.
__device__ inline void to_columns(f32x16 &c)
{
#pragma unroll
    for (int q = 0; q < 4; q += 2)
#pragma unroll
        for (int r = 0; r < 4; ++r)
        {
            const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(c[4 * q + r]), __float_as_uint(c[4 * q + 4 + r]), false, false);
            c[4 * q + r]     = __uint_as_float(s[0]);
            c[4 * q + 4 + r] = __uint_as_float(s[1]);
        }
}

struct GemmArgs
{
    Panel a, b;       // C[i][j] = sum over the contraction of a[i][.] b[j][.]
    int nkb;          // contraction blocks multiplied: even (panels are padded to fours, with zeros)
    int tiles_m, tiles_n;
    int symmetric;    // only tiles with tile row <= tile column
    int splits, split_kb;  // the contraction in `splits` runs of split_kb blocks (even), a workgroup each
    int batch;
    int64_t a_batch, b_batch;  // bytes from one product's operands to the next one's
    int xcds;
    int64_t blocks() const
    {
        return (int64_t)batch * splits * (symmetric ? (int64_t)tiles_m * (tiles_m + 1) / 2 : (int64_t)tiles_m * tiles_n);
    }
};

// Which tile a workgroup computes. Workgroups are dealt to the XCDs in turn, and each XCD has an L2 of its own: the tiles are
// cut into one run per XCD, and inside a run they go down groups of four tile rows, so that what an XCD holds at a time is a
// compact rectangle whose operands it reads once.
__device__ inline void tile_of(const GemmArgs &g, int &z, int &split, int &tm, int &tn)
{
    const unsigned total = gridDim.x, xcds = (unsigned)g.xcds, bid = blockIdx.x;
    const unsigned x = bid % xcds, q = total / xcds, rem = total % xcds;
    unsigned t = x * q + (x < rem ? x : rem) + bid / xcds;
    const unsigned per = g.symmetric ? (unsigned)g.tiles_m * (g.tiles_m + 1) / 2 : (unsigned)g.tiles_m * g.tiles_n;
    z = 0, split = 0;
    if (t >= per)
    {
        const unsigned run = t / per;
        t -= run * per;
        z = (int)(run / (unsigned)g.splits), split = (int)(run - (unsigned)z * g.splits);
    }
    if (g.symmetric)
    {
        int j = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
        while ((unsigned)j * (j + 1) / 2 > t)
            --j;
        while ((unsigned)(j + 1) * (j + 2) / 2 <= t)
            ++j;
        tn = j, tm = (int)(t - (unsigned)j * (j + 1) / 2);
        return;
    }
    const unsigned gsz = 4u * g.tiles_n, grp = t / gsz, in = t - grp * gsz, first = grp * 4;
    const unsigned rows = min(4u, (unsigned)g.tiles_m - first);
    tm = (int)(first + in % rows), tn = (int)(in / rows);
}

// What an epilogue is handed: its accumulators stay in the kernel, one call per workgroup.
template <int BM, int BN, int WM, int WN>
struct Tile
{
    static constexpr int MI = BM / 32 / WM, NI = BN / 32 / WN;
    static constexpr int kRows = BM, kCols = BN, kWavesM = WM, kWavesN = WN;
    int z, split, tm, tn;  // product, run of the contraction, tile row, tile column
    int wm, wn, lane;  // wave's place in the tile
    char *lds;         // the stages' LDS, free for the epilogue (every wave has passed a barrier)
    __device__ int64_t row_block(int mi) const { return (int64_t)tm * (BM / 32) + wm * MI + mi; }
    __device__ int64_t col_block(int ni) const { return (int64_t)tn * (BN / 32) + wn * NI + ni; }
    __device__ float *wave_scratch() const  // 32 rows of 33 floats per wave
    {
        return reinterpret_cast<float *>(lds) + (wm * WN + wn) * (32 * 33);
    }
};

template <int BM, int BN, int WM, int WN, class Epilogue>
__global__ __launch_bounds__(64 * WM *WN, 2) void split_gemm_kernel(const GemmArgs g, const Epilogue epilogue)
{
    using T = Tile<BM, BN, WM, WN>;
    constexpr int NW = WM * WN, MI = T::MI, NI = T::NI;
    constexpr int kUnits = (BM + BN) / 32 * 2;  // KB of a stage: one load instruction of one wave each
    static_assert(kUnits % NW == 0 && BM % (32 * WM) == 0 && BN % (32 * WN) == 0, "waves share a stage evenly");
    constexpr int L = kUnits / NW;
    constexpr int kStageBytes = kUnits * 1024;
    static_assert(NW * 32 * 33 * 4 <= kStages * kStageBytes, "the epilogue's scratch lies in the stages");
    __shared__ __attribute__((aligned(1024))) char lds[kStages * kStageBytes];

    T t;
    tile_of(g, t.z, t.split, t.tm, t.tn);
    const int kb0 = t.split * g.split_kb, nkb = min(g.split_kb, g.nkb - kb0);
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    t.lane = threadIdx.x & 63, t.wm = wave / WN, t.wn = wave % WN, t.lds = lds;

    // the wave's share of a stage: L half blocks, A's before B's
    constexpr int kUnitsA = BM / 32 * 2;
    const char *a_base = g.a.base + t.z * g.a_batch + t.tm * (BM / 32) * g.a.row_block_bytes() + (int64_t)kb0 * kBlockBytes;
    const char *b_base = g.b.base + t.z * g.b_batch + t.tn * (BN / 32) * g.b.row_block_bytes() + (int64_t)kb0 * kBlockBytes;
    const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    const unsigned lane_off = t.lane * 16;
    i32x4 rsrc[L];
    unsigned unit_off[L];
#pragma unroll
    for (int i = 0; i < L; ++i)
    {
        const int u = wave * L + i;
        const bool for_a = u < kUnitsA;
        const int v = for_a ? u : u - kUnitsA;
        rsrc[i]     = buffer_of(for_a ? a_base : b_base);
        unit_off[i] = (unsigned)((v >> 1) * (for_a ? g.a.row_block_bytes() : g.b.row_block_bytes())) + (unsigned)(v & 1) * 1024;
    }
    // the wave's part of stage kb into its slot; past the last block the last one is loaded again (read by no product),
    // so that the count of queued loads is the same in every round
    auto queue = [&](int kb) {
        const unsigned dst = lds0 + (unsigned)(kb % kStages) * kStageBytes + (unsigned)(wave * L) * 1024;
        const unsigned at  = (unsigned)min(kb, nkb - 1) * kBlockBytes;
#pragma unroll
        for (int i = 0; i < L; ++i)
            load_to_lds_16(rsrc[i], dst + i * 1024, lane_off, unit_off[i] + at);
    };
    // fragments: B's of a whole stage, A's one block at a time (registers: 2 x 16 + 2 x 8 beside 128 accumulators)
    struct FragsB
    {
        half8 h[NI], l[NI];
    };
    struct FragA
    {
        half8 h, l;
    };
    auto read_b = [&](int kb, FragsB &f) {
        const char *slot = lds + (kb % kStages) * kStageBytes + lane_off + (BM / 32 + t.wn * NI) * kBlockBytes;
#pragma unroll
        for (int i = 0; i < NI; ++i)
        {
            f.h[i] = *reinterpret_cast<const half8 *>(slot + i * kBlockBytes);
            f.l[i] = *reinterpret_cast<const half8 *>(slot + i * kBlockBytes + 1024);
        }
    };
    auto read_a = [&](int kb, int i, FragA &f) {
        const char *slot = lds + (kb % kStages) * kStageBytes + lane_off + (t.wm * MI + i) * kBlockBytes;
        f.h = *reinterpret_cast<const half8 *>(slot);
        f.l = *reinterpret_cast<const half8 *>(slot + 1024);
    };
    f32x16 acc[MI][NI];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                acc[i][j][e] = 0.f;
    constexpr bool kApart = BM * BN < 256 * 256;
    f32x16 cross[kApart ? MI : 1][kApart ? NI : 1];
    if constexpr (kApart)
    {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    cross[i][j][e] = 0.f;
    }
    // One stage. A's next fragment is read under the products of the present one; before the last block's products comes the
    // round's only barrier: every wave has read all of stage kb, whose slot takes stage kb + kStages, and stage kb + 1 has
    // landed, whose first fragments are read under those products. P: which of the two A fragments the stage begins with.
    FragA fa[2];
    FragsB fb[2];
    auto stage = [&](int kb, auto parity) {
        constexpr int P = decltype(parity)::value, A0 = (P * MI) & 1;
#pragma unroll
        for (int i = 0; i < MI; ++i)
        {
            if (i + 1 < MI)
                read_a(kb, i + 1, fa[(A0 + i + 1) & 1]);
            else
            {
                wait_loads_and_lds<L *(kStages - 2)>();
                barrier();
                queue(kb + kStages);
                read_b(kb + 1, fb[P ^ 1]);
                read_a(kb + 1, 0, fa[(A0 + i + 1) & 1]);
            }
            __builtin_amdgcn_sched_barrier(0);
            const FragA &a = fa[(A0 + i) & 1];
#pragma unroll
            for (int j = 0; j < NI; ++j)
            {
                f32x16 &c = kApart ? cross[kApart ? i : 0][kApart ? j : 0] : acc[i][j];
                c         = __builtin_amdgcn_mfma_f32_32x32x16_f16(a.h, fb[P].l[j], c, 0, 0, 0);
            }
#pragma unroll
            for (int j = 0; j < NI; ++j)
            {
                f32x16 &c = kApart ? cross[kApart ? i : 0][kApart ? j : 0] : acc[i][j];
                c         = __builtin_amdgcn_mfma_f32_32x32x16_f16(a.l, fb[P].h[j], c, 0, 0, 0);
            }
#pragma unroll
            for (int j = 0; j < NI; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a.h, fb[P].h[j], acc[i][j], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    for (int s = 0; s < kStages; ++s)
        queue(s);
    wait_loads_and_lds<L *(kStages - 1)>();
    barrier();
    read_b(0, fb[0]);
    read_a(0, 0, fa[0]);
    for (int kb = 0; kb < nkb; kb += 2)
    {
        stage(kb, std::integral_constant<int, 0>{});
        stage(kb + 1, std::integral_constant<int, 1>{});
    }
    wait_loads_and_lds<0>();  // no load is under way into LDS that the epilogue writes
    barrier();
    if constexpr (kApart)
    {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    acc[i][j][e] += cross[i][j][e];
    }
    epilogue(t, acc);
}

// The product for few tiles: a workgroup of four waves holds a 64 x 64 tile, each wave the whole tile for every fourth
// contraction block. No wave reads what another one does, so fragments come straight from memory into registers, without LDS,
// barriers or waits for each other; the four partial sums meet in LDS at the end, added in the waves' order.
constexpr int kDirectWaves = 4;

template <class Epilogue>
__global__ __launch_bounds__(64 * kDirectWaves, 2) void split_gemm_direct_kernel(const GemmArgs g, const Epilogue epilogue)
{
    __shared__ __attribute__((aligned(16))) char lds[kDirectWaves * 4 * 4096];
    Tile<64, 64, 2, 2> t;
    tile_of(g, t.z, t.split, t.tm, t.tn);
    const int kb0 = t.split * g.split_kb, nkb = min(g.split_kb, g.nkb - kb0);
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    t.lane = threadIdx.x & 63, t.lds = lds;
    const int64_t a_rb = g.a.row_block_bytes(), b_rb = g.b.row_block_bytes();
    const auto ra = __builtin_amdgcn_make_buffer_rsrc(g.a.base + t.z * g.a_batch + t.tm * 2 * a_rb + (int64_t)kb0 * kBlockBytes, 0, 0x7fffffff, 0x00020000);
    const auto rb = __builtin_amdgcn_make_buffer_rsrc(g.b.base + t.z * g.b_batch + t.tn * 2 * b_rb + (int64_t)kb0 * kBlockBytes, 0, 0x7fffffff, 0x00020000);
    struct Frags
    {
        half8 ah[2], al[2], bh[2], bl[2];
    };
    const auto load = [&](int kb, Frags &f) {
        // past the last block the offset lies past the buffer, and zeros arrive
        const unsigned off = kb < nkb ? (unsigned)kb * kBlockBytes + t.lane * 16 : 0x80000000u;
#pragma unroll
        for (int i = 0; i < 2; ++i)
        {
            f.ah[i] = __builtin_bit_cast(half8, __builtin_amdgcn_raw_buffer_load_b128(ra, off, (int)(i * a_rb), 0));
            f.al[i] = __builtin_bit_cast(half8, __builtin_amdgcn_raw_buffer_load_b128(ra, off, (int)(i * a_rb) + 1024, 0));
            f.bh[i] = __builtin_bit_cast(half8, __builtin_amdgcn_raw_buffer_load_b128(rb, off, (int)(i * b_rb), 0));
            f.bl[i] = __builtin_bit_cast(half8, __builtin_amdgcn_raw_buffer_load_b128(rb, off, (int)(i * b_rb) + 1024, 0));
        }
    };
    f32x16 acc[2][2], cross[2][2];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e)
            acc[i >> 1][i & 1][e] = cross[i >> 1][i & 1][e] = 0.f;
    const auto multiply = [&](const Frags &f) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                cross[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.ah[i], f.bl[j], cross[i][j], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                cross[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.al[i], f.bh[j], cross[i][j], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.ah[i], f.bh[j], acc[i][j], 0, 0, 0);
    };
    Frags f0, f1;
    load(wave, f0);
    load(wave + kDirectWaves, f1);
    for (int kb = wave; kb < nkb; kb += 2 * kDirectWaves)
    {
        multiply(f0);
        load(kb + 2 * kDirectWaves, f0);
        multiply(f1);
        load(kb + 3 * kDirectWaves, f1);
    }
    f32x4 *mine = reinterpret_cast<f32x4 *>(lds) + wave * 4 * 256 + t.lane;
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int q = 0; q < 4; ++q)
        {
            const f32x16 c = acc[b >> 1][b & 1] + cross[b >> 1][b & 1];
            mine[b * 256 + q * 64] = f32x4{c[4 * q], c[4 * q + 1], c[4 * q + 2], c[4 * q + 3]};
        }
    __syncthreads();
    // wave b finishes block b
    t.wm = (wave >> 1) & 1, t.wn = wave & 1;
    f32x16 sum[1][1];
    {
        const f32x4 *theirs = reinterpret_cast<const f32x4 *>(lds) + wave * 256 + t.lane;
#pragma unroll
        for (int q = 0; q < 4; ++q)
        {
            f32x4 s = theirs[q * 64];
#pragma unroll
            for (int w = 1; w < kDirectWaves; ++w)
                s += theirs[w * 4 * 256 + q * 64];
            sum[0][0][4 * q] = s[0], sum[0][0][4 * q + 1] = s[1], sum[0][0][4 * q + 2] = s[2], sum[0][0][4 * q + 3] = s[3];
        }
    }
    __syncthreads();  // the epilogue writes LDS
    epilogue(t, sum);
}

// How a product is cut: tile and runs of the contraction.
struct Cut
{
    int bm, bn, splits;
    int split_kb;
};

// The cut with the least estimated time. Measured on an MI355X: microseconds per contraction block (16 values) of a tile alone
// on its compute unit and of one among as many as fit there (256 x 256 and its halves: one; the others two), the rate in
// TFLOP/s at which many of them run into the chip's power limit (long symmetric products lower: their tiles share less),
// and microseconds a round of tiles spends outside its loop. Large tiles read their operands less often and leave compute
// units idle in a short last round. Runs of the contraction (may_split) cost a pass over the partial results: out_bytes
// written per run, read once. exact: only tiles with accumulators apart for the cross terms. For example 4096 x 4096 x 4096:
// 323 us with 256 x 256, 325 with 256 x 128, 333 with 128 x 128, 404 with 64 x 64; 1024 x 1024 x 1024: 52, 29, 19 and 8.6 us.
// A short last round of tiles is left as it is: computed as smaller tiles in runs (4096 x 4096 symmetric products, 16 of 528
// tiles) it saved nothing, because a chip at its power limit makes up for idle compute units with its clock.
inline Cut pick_cut(int64_t rows_pad, int64_t cols_pad, bool symmetric, int64_t batch, int nkb, bool may_split = false, double out_bytes = 0,
                    bool exact = false)
{
    struct Option
    {
        int bm, bn, resident;
        double alone, full, rate, symmetric_rate, fixed;
    };
    static const Option options[] = {{256, 256, 1, 0.80, 0.80, 425, 425, 12.0}, {256, 128, 1, 0.46, 0.46, 405, 405, 7.0},
                                     {128, 256, 1, 0.46, 0.46, 405, 405, 7.0}, {128, 128, 2, 0.37, 0.26, 400, 400, 4.0},
                                     {64, 64, 2, 0.107, 0.085, 330, 230, 2.0}};
    const int cus = device_cus();
    Cut best{64, 64, 1, nkb};
    double best_cost = 0;
    for (const Option &o : options)
    {
        if (rows_pad % o.bm || cols_pad % o.bn || (symmetric && o.bm != o.bn) || (exact && o.bm * o.bn == 256 * 256))
            continue;
        const int64_t tm = rows_pad / o.bm, tn = cols_pad / o.bn, tiles = batch * (symmetric ? tm * (tm + 1) / 2 : tm * tn);
        for (int s = 1; s <= (may_split ? 32 : 1) && (s == 1 || nkb / s >= 8); ++s)
        {
            const int kb = s == 1 ? nkb : (int)ceil_div(nkb, 2 * s) * 2;
            if (s > 1 && (int64_t)(s - 1) * kb >= nkb)
                continue;
            const int64_t work = tiles * s, slots = (int64_t)cus * o.resident, full = work / slots, rest = work - full * slots;
            const double last = rest == 0 ? 0.0 : rest <= cus ? o.alone : o.full * (double)ceil_div(rest, cus);
            double cost = kb * ((double)full * o.resident * o.full + last);
            cost = std::max(cost, (double)work * kb * o.bm * o.bn * 32.0 / (symmetric ? o.symmetric_rate : o.rate) / 1e6) + o.fixed * (double)(full + (rest != 0));
            if (s > 1)
                cost += 5.0 + out_bytes * (s + 1) / 4e6;
            if (best_cost == 0 || cost < best_cost)
                best = Cut{o.bm, o.bn, s, kb}, best_cost = cost;
        }
    }
    return best;
}

// Where a run of the contraction leaves its accumulators: [product][row block][column block][run], 32 x 32 each as a wave
// holds them.
struct PartEpilogue
{
    f32x4 *parts;
    int64_t row_blocks, col_blocks;
    int splits;
    __device__ f32x4 *at(int z, int64_t rb, int64_t cb) const { return parts + ((z * row_blocks + rb) * col_blocks + cb) * splits * 256; }
    template <class T, class Acc>
    __device__ void operator()(const T &t, Acc &acc) const
    {
#pragma unroll
        for (int mi = 0; mi < T::MI; ++mi)
#pragma unroll
            for (int ni = 0; ni < T::NI; ++ni)
            {
                const f32x16 &c = acc[mi][ni];
                f32x4 *out      = at(t.z, t.row_block(mi), t.col_block(ni)) + t.split * 256 + t.lane;
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    out[q * 64] = f32x4{c[4 * q], c[4 * q + 1], c[4 * q + 2], c[4 * q + 3]};
            }
    }
};

// The runs' accumulators added up in order, then the epilogue: the second launch of a product whose contraction is cut, on
// 64 x 64 tiles whatever the first one's were (many workgroups, each a short chain of loads).
template <class Epilogue>
__global__ __launch_bounds__(256) void split_gemm_finish_kernel(const GemmArgs g, const PartEpilogue parts, const Epilogue epilogue)
{
    __shared__ __attribute__((aligned(16))) char lds[4 * 32 * 33 * 4];
    Tile<64, 64, 2, 2> t;
    tile_of(g, t.z, t.split, t.tm, t.tn);
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    t.lane = threadIdx.x & 63, t.wm = wave >> 1, t.wn = wave & 1, t.lds = lds;
    const f32x4 *in = parts.at(t.z, t.row_block(0), t.col_block(0)) + t.lane;
    f32x16 acc[1][1];
#pragma unroll
    for (int e = 0; e < 16; ++e)
        acc[0][0][e] = 0.f;
#pragma unroll 8
    for (int s = 0; s < parts.splits; ++s)
#pragma unroll
        for (int q = 0; q < 4; ++q)
        {
            const f32x4 v = in[s * 256 + q * 64];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                acc[0][0][4 * q + e] += v[e];
        }
    epilogue(t, acc);
}

// bytes of the runs' accumulators
inline size_t part_bytes(const Cut &cut, int64_t rows_pad, int64_t cols_pad, int64_t batch)
{
    return cut.splits > 1 ? (size_t)cut.splits * (size_t)(batch * rows_pad * cols_pad) * 4 : 0;
}

template <class Epilogue>
inline int launch_tiles(const GemmArgs &g, const Cut &cut, const Epilogue &e, hipStream_t st)
{
    const int64_t blocks = g.blocks();
    const int threads    = cut.bm * cut.bn > 128 * 128 ? 512 : 256;
    ODL_REQUIRE(blocks <= ((int64_t)1 << 32) / threads - 1, "product of too many tiles");
    if (blocks == 0 || g.nkb == 0)
        return fail(ODL_ERR_RUNTIME, "empty product");
    const dim3 grid((unsigned)blocks);
    if (cut.bm == 256 && cut.bn == 256)
        split_gemm_kernel<256, 256, 2, 4, Epilogue><<<grid, dim3(512), 0, st>>>(g, e);
    else if (cut.bm == 256)
        split_gemm_kernel<256, 128, 4, 2, Epilogue><<<grid, dim3(512), 0, st>>>(g, e);
    else if (cut.bn == 256)
        split_gemm_kernel<128, 256, 2, 4, Epilogue><<<grid, dim3(512), 0, st>>>(g, e);
    else if (cut.bm == 128)
        split_gemm_kernel<128, 128, 2, 2, Epilogue><<<grid, dim3(256), 0, st>>>(g, e);
    else
        split_gemm_direct_kernel<Epilogue><<<grid, dim3(64 * kDirectWaves), 0, st>>>(g, e);
    ODL_LAUNCH_CHECK();
    return ODL_OK;
}

inline GemmArgs cut_args(GemmArgs g, int64_t rows_pad, int64_t cols_pad, const Cut &cut)
{
    g.tiles_m = (int)(rows_pad / cut.bm), g.tiles_n = (int)(cols_pad / cut.bn), g.xcds = chip().xcds;
    g.splits = cut.splits, g.split_kb = cut.split_kb;
    return g;
}

// the epilogue sees t.split, the run of the contraction its accumulators cover
template <class Epilogue>
inline int launch_gemm(const GemmArgs &g, int64_t rows_pad, int64_t cols_pad, const Cut &cut, const Epilogue &e, hipStream_t st)
{
    return launch_tiles(cut_args(g, rows_pad, cols_pad, cut), cut, e, st);
}

// the epilogue sees the whole sums: with runs of the contraction (parts: part_bytes) in a second launch
template <class Epilogue>
inline int launch_whole_gemm(const GemmArgs &args, int64_t rows_pad, int64_t cols_pad, const Cut &cut, void *parts, const Epilogue &e, hipStream_t st)
{
    GemmArgs g = cut_args(args, rows_pad, cols_pad, cut);
    if (cut.splits == 1)
        return launch_tiles(g, cut, e, st);
    const PartEpilogue p{static_cast<f32x4 *>(parts), rows_pad / 32, cols_pad / 32, cut.splits};
    if (int rc = launch_tiles(g, cut, p, st))
        return rc;
    g = cut_args(args, rows_pad, cols_pad, Cut{64, 64, 1, args.nkb});
    const int64_t blocks = g.blocks();
    ODL_REQUIRE(blocks <= ((int64_t)1 << 32) / 256 - 1, "product of too many tiles");
    split_gemm_finish_kernel<Epilogue><<<dim3((unsigned)blocks), dim3(256), 0, st>>>(g, p, e);
    ODL_LAUNCH_CHECK();
    return ODL_OK;
}

// Values [rows, cols] into panels: `r` has the matrix's rows as rows, `t` its columns (either may have a null base). Src gives
// the value at (row, col) in bounds, and factor() what all are multiplied by (every thread calls it once, when its values are
// under way: it may take its own time); a workgroup of 256 threads takes 64 x 64 values through LDS. Rows and
// columns up to the padded extents are written as zeros.
template <class Src, class Factor>
__device__ inline void split_tile(const Src &src, const Factor &factor, int64_t rows, int64_t cols, int64_t r0, int64_t c0, const Panel &r, const Panel &t,
                                  float (*tile)[65])
{
    const int tid = threadIdx.x;
    {
        const int c = tid & 63;
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i)
        {
            const int64_t row = r0 + (tid >> 6) + 4 * i, col = c0 + c;
            v[i] = row < rows && col < cols ? src(row, col) : 0.f;
        }
        const auto by = factor();
#pragma unroll
        for (int i = 0; i < 16; ++i)
            tile[(tid >> 6) + 4 * i][c] = (float)(v[i] * by);
    }
    __syncthreads();
    const int lane = tid & 63;
#pragma unroll
    for (int f = tid >> 6; f < 8; f += 4)  // fragments: 2 row blocks x 4 contraction blocks
    {
        const int rb = f >> 2, kb = f & 3;
        float v[8];
        if (r.base)
        {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                v[e] = tile[rb * 32 + (lane & 31)][kb * 16 + (lane >> 5) * 8 + e];
            store_fragment(r, r0 / 32 + rb, c0 / 16 + kb, lane, v);
        }
        if (t.base)
        {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                v[e] = tile[kb * 16 + (lane >> 5) * 8 + e][rb * 32 + (lane & 31)];
            store_fragment(t, c0 / 32 + rb, r0 / 16 + kb, lane, v);
        }
    }
}
}  // namespace split
}  // namespace odl
