// mx_gemm.hip -- products of MXFP4 activations and MXFP4 weights on the scaled matrix cores (layouts: mx.hpp):
//
//   qmm_gemv_mxfp4       y[m][n] = W[n] . x[m], m < 64: decode and draft verification
//   qmm_gemv_moe_mxfp4   the same for the routed experts of up to 16 tokens, by ids
//   qmm_gemm_mxfp4       any number of rows: prompts
//   qmm_moe_gemm_mxfp4   rows sorted by expert (qmm_moe_sort)
//
// A scaled matrix instruction multiplies weight rows by activation rows with their block scales and adds to
// f32: 16 x 16 over 128 values in the GEMV (few rows), 32 x 32 over 64 in the GEMM (6.4 PFLOP/s measured from
// registers against 5.4 for the former: it reads half the operand bytes per product).  The weight is the first
// operand, so a lane ends with four successive outputs of one activation row.
//
// Order of sums.  GEMM: an output is one chain of instructions over K, whatever the tile, M or N.  GEMV: K's groups of four steps are cut into S contiguous runs, S chosen by K alone; each run is one chain
// and the S sums are added in order.  So an output's bits depend on its own rows and K, not on the call.
#include "mx_tile.hpp"

#include <cmath>

namespace qmm {
namespace {

// ------------------------------------------------------------------------------------------
// GEMV.  A workgroup is one strip (16 weight rows), its S waves the runs of K: a weight byte is read once, by
// contiguous kilobytes, straight into the operand registers, two groups (8 KB a wave) ahead.
constexpr int kGemvMaxWaves = 8, kGemvMaxRows = 64;

// S for G groups: one wave a group up to 8, else the count of 4 .. 8 that leaves the least imbalance
int gemv_waves(int G) {
    if (G <= kGemvMaxWaves) return G;
    int best = 4;
    for (int s = 5; s <= kGemvMaxWaves; ++s)
        if ((G + s - 1) / s * s <= (G + best - 1) / best * best) best = s;
    return best;
}

template <int MF>
struct GemvGroup {
    uint4 w[4], a[MF][4];
    uint32_t ws, as[MF][4];
};

template <int MF>
__device__ __forceinline__ void gemv_load(GemvGroup<MF>& r, const uint8_t* strip, const uint8_t* const (&qr)[MF], const uint8_t* const (&er)[MF],
                                          int g, int K128, int lane) {
    const uint8_t* ws = strip + (uint32_t)K128 * 1024u;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const uint32_t kt = (uint32_t)min(4 * g + s, K128 - 1);      // a short last group re-reads its last step, unused
        r.w[s] = ld16(strip + kt * 1024u + lane * 16);
    }
    r.ws = *(const uint32_t*)(ws + (uint32_t)g * 256u + lane * 4);
#pragma unroll
    for (int f = 0; f < MF; ++f)
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const uint32_t kt = (uint32_t)min(4 * g + s, K128 - 1);
            r.a[f][s] = ld16(qr[f] + kt * 64u);
            r.as[f][s] = er[f][kt * 4u];
        }
}

template <int MF>
__device__ __forceinline__ void gemv_mul(const GemvGroup<MF>& r, mx_v4f (&acc)[MF], int g, int K128) {
    const int n = K128 - 4 * g;                          // steps left (uniform)
#pragma unroll
    for (int f = 0; f < MF; ++f) acc[f] = mx_mfma<0>(r.w[0], r.a[f][0], acc[f], r.ws, r.as[f][0]);
    if (n > 1) {
#pragma unroll
        for (int f = 0; f < MF; ++f) acc[f] = mx_mfma<1>(r.w[1], r.a[f][1], acc[f], r.ws, r.as[f][1]);
    }
    if (n > 2) {
#pragma unroll
        for (int f = 0; f < MF; ++f) acc[f] = mx_mfma<2>(r.w[2], r.a[f][2], acc[f], r.ws, r.as[f][2]);
    }
    if (n > 3) {
#pragma unroll
        for (int f = 0; f < MF; ++f) acc[f] = mx_mfma<3>(r.w[3], r.a[f][3], acc[f], r.ws, r.as[f][3]);
    }
}

// this wave's run of K for activation rows row[f] (per lane: row of lane % 16)
template <int MF>
__device__ __forceinline__ void gemv_run(const uint8_t* strip, qmm_xmx x, const int (&row)[MF], int K128, int S, int wave, mx_v4f (&acc)[MF]) {
    const int lane = threadIdx.x & 63, blk = lane >> 4, G = mx_groups(K128);
    const int g0 = wave * G / S, g1 = (wave + 1) * G / S;
    const uint8_t* qr[MF];
    const uint8_t* er[MF];
#pragma unroll
    for (int f = 0; f < MF; ++f) {
        qr[f] = x.q + (size_t)row[f] * K128 * 64 + blk * 16;
        er[f] = x.e + (size_t)row[f] * K128 * 4 + blk;
        acc[f] = mx_v4f{0.f, 0.f, 0.f, 0.f};
    }
    GemvGroup<MF> r0, r1;
    if (g0 < g1) gemv_load<MF>(r0, strip, qr, er, g0, K128, lane);
    for (int g = g0; g < g1; g += 2) {
        if (g + 1 < g1) gemv_load<MF>(r1, strip, qr, er, g + 1, K128, lane);
        gemv_mul<MF>(r0, acc, g, K128);
        if (g + 1 < g1) {
            if (g + 2 < g1) gemv_load<MF>(r0, strip, qr, er, g + 2, K128, lane);
            gemv_mul<MF>(r1, acc, g + 1, K128);
        }
    }
}

// the S runs' sums, added in order: thread i of the workgroup gets item i = 64 f + lane
template <int MF>
__device__ __forceinline__ void gemv_reduce(mx_v4f* red, const mx_v4f (&acc)[MF], int wave) {
#pragma unroll
    for (int f = 0; f < MF; ++f) red[(wave * MF + f) * 64 + (threadIdx.x & 63)] = acc[f];
    __syncthreads();
}
template <int MF>
__device__ __forceinline__ mx_v4f gemv_sum(const mx_v4f* red, int i, int S) {
    mx_v4f v = red[i];
    for (int w = 1; w < S; ++w) v += red[w * MF * 64 + i];
    return v;
}

template <int MF, bool BF>
__global__ void __launch_bounds__(64 * kGemvMaxWaves) k_gemv_mxfp4(const uint8_t* __restrict__ W, qmm_xmx x, void* __restrict__ y, int N, int K128,
                                                                   int ncol, int vec) {
    extern __shared__ __align__(16) uint8_t smem[];
    mx_v4f* red = (mx_v4f*)smem;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), S = blockDim.x >> 6;
    const uint8_t* strip = W + (size_t)blockIdx.x * mx_strip_bytes(K128);
    int row[MF];
#pragma unroll
    for (int f = 0; f < MF; ++f) row[f] = min(16 * f + (lane & 15), ncol - 1);
    mx_v4f acc[MF];
    gemv_run<MF>(strip, x, row, K128, S, wave, acc);
    gemv_reduce<MF>(red, acc, wave);
    for (int i = threadIdx.x; i < 64 * MF; i += blockDim.x) {
        const mx_v4f v = gemv_sum<MF>(red, i, S);
        const int m = 16 * (i >> 6) + (i & 15), n = (int)blockIdx.x * 16 + 4 * ((i >> 4) & 3);
        if (m < ncol && n < N) mx_store4<BF>(y, (size_t)m * N + n, v, N - n, vec);
    }
}

// Experts by ids: workgroup (strip, slot).  The first slot of an expert computes all slots that hold it, 16 at
// a time (a token lists an expert once, so 16 tokens make one pass), the others leave: an expert is read once.
constexpr int kMoeGemvMaxT = 16, kMoeGemvMaxSlots = kMoeGemvMaxT * kMoeMaxSlots;

template <bool BF>
__global__ void __launch_bounds__(64 * kGemvMaxWaves) k_gemv_moe_mxfp4(const uint8_t* __restrict__ W, const uint8_t* __restrict__ Wsh, size_t ebytes,
                                                                       const int* __restrict__ ids, qmm_xmx x, void* __restrict__ y, int nslots,
                                                                       int per_token, int xrow_te, int nexp, int N, int K128, int vec) {
    extern __shared__ __align__(16) uint8_t smem[];
    mx_v4f* red = (mx_v4f*)smem;
    __shared__ int cols[kMoeGemvMaxSlots];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), S = blockDim.x >> 6;
    const int te = blockIdx.y;
    // an id below 0 is the shared expert (expert 0 without one), one beyond the last is the last
    const int first = Wsh ? -1 : 0;
    const int id = min(max(ids[te], first), nexp - 1);
    int n = 0;
    for (int base = 0; base < nslots; base += 64) {      // every wave finds the same list
        const int sl = base + lane;
        const bool same = sl < nslots && min(max(ids[min(sl, nslots - 1)], first), nexp - 1) == id;
        const uint64_t hit = __builtin_amdgcn_ballot_w64(same);
        if (base <= te && hit) {
            const int lead = base + __builtin_ctzll(hit);
            if (lead < te) return;                       // uniform over the workgroup
        }
        if (same && wave == 0) cols[n + __builtin_popcountll(hit & ((1ull << lane) - 1))] = sl;
        n += __builtin_popcountll(hit);
    }
    __syncthreads();
    const uint8_t* strip = (id < 0 ? Wsh : W + (size_t)id * ebytes) + (size_t)blockIdx.x * mx_strip_bytes(K128);
    for (int c0 = 0; c0 < n; c0 += 16) {
        const int slot = cols[min(c0 + (lane & 15), n - 1)];
        const int row[1] = {xrow_te ? slot : slot / per_token};
        mx_v4f acc[1];
        gemv_run<1>(strip, x, row, K128, S, wave, acc);
        gemv_reduce<1>(red, acc, wave);
        if (threadIdx.x < 64) {
            const mx_v4f v = gemv_sum<1>(red, threadIdx.x, S);
            const int m = c0 + (lane & 15), nn = (int)blockIdx.x * 16 + 4 * (lane >> 4);
            if (m < n && nn < N) mx_store4<BF>(y, (size_t)slot * N + nn, v, N - nn, vec);
        }
        __syncthreads();                                 // red is written again
    }
}

// ------------------------------------------------------------------------------------------
// GEMM.  Workgroup i runs on XCD i % 8: each XCD takes a contiguous range of tiles, rows fastest, so that the tiles
// it runs together share weight strips in its L2.
__device__ __forceinline__ uint32_t xcd_tile() {
    const uint32_t total = gridDim.x, xcd = blockIdx.x & 7, q = total >> 3, rem = total & 7;
    return xcd * q + min(xcd, rem) + (blockIdx.x >> 3);
}

template <int MF, int NF, int D, int PER, bool BF>
__global__ void __launch_bounds__(256, PER) k_gemm_mxfp4_reg(const uint8_t* __restrict__ W, qmm_xmx x, void* __restrict__ Dst, int M, int N, int K128,
                                                             int mtiles, int vec) {
    using T = MxReg<MF, NF>;
    extern __shared__ __align__(16) uint8_t smem[];
    const uint32_t t = xcd_tile();
    const int m0 = (int)(t % (uint32_t)mtiles) * T::kRows, n0 = (int)(t / (uint32_t)mtiles) * T::kCols;
    mx_v16f acc[NF][MF];
    mx_tile_reg<MF, NF, D, PER == 1>(smem, W, x, n0 / 16, (N + 15) / 16, K128, [&](int r) { return min(m0 + r, M - 1); }, acc);
    mx_store<MF, NF, BF>(smem, acc, Dst, n0 + 32 * NF * (int)(threadIdx.x >> 6), N, vec, [&](int r) { return m0 + r < M ? (int64_t)(m0 + r) : -1; });
}

template <int MF, int NF, int NS, bool BF>
__global__ void __launch_bounds__(512, 2) k_gemm_mxfp4_dma(const uint8_t* __restrict__ W, qmm_xmx x, void* __restrict__ Dst, int M, int N, int K128,
                                                           int mtiles, int vec) {
    using T = MxDma<MF, NF, NS>;
    extern __shared__ __align__(16) uint8_t smem[];
    const uint32_t t = xcd_tile();
    const int m0 = (int)(t % (uint32_t)mtiles) * T::kRows, n0 = (int)(t / (uint32_t)mtiles) * T::kCols;
    mx_v16f acc[NF][MF];
    mx_tile_dma<MF, NF, NS>(smem, W, x, n0 / 16, (N + 15) / 16, K128, [&](int r) { return min(m0 + r, M - 1); }, acc);
    const int wave = threadIdx.x >> 6, mw = m0 + 32 * MF * (wave >> 2);
    mx_store<MF, NF, BF>(smem, acc, Dst, n0 + 32 * NF * (wave & 3), N, vec, [&](int r) { return mw + r < M ? (int64_t)(mw + r) : -1; });
}

// Grouped: workgroup (tile of one expert's rows, block of 128 outputs); a tile's rows 64 at a time, with as
// many 32-row fragments as they need.
constexpr int kMoeNF = 1, kMoeD = 8, kMoeCols = 128 * kMoeNF, kMoeRows = 64;

template <int MF, bool BF>
__device__ __forceinline__ void moe_rows(uint8_t* smem, const uint8_t* We, qmm_xmx x, const int* rowtab, int k0, int n, int n0, void* D, int N, int K128,
                                         int vec) {
    mx_v16f acc[kMoeNF][MF];
    mx_tile_reg<MF, kMoeNF, kMoeD, false>(smem, We, x, n0 / 16, (N + 15) / 16, K128, [&](int r) {
        const int k = k0 + min(r, n - 1);
        return rowtab ? rowtab[k] : k;
    }, acc);
    mx_store<MF, kMoeNF, BF>(smem, acc, D, n0 + 32 * kMoeNF * (int)(threadIdx.x >> 6), N, vec, [&](int r) { return r < n ? (int64_t)(k0 + r) : -1; });
}

template <bool BF>
__global__ void __launch_bounds__(256, 2) k_moe_gemm_mxfp4(const uint8_t* __restrict__ W, const uint8_t* __restrict__ Wsh, size_t ebytes,
                                                           const qmm_moe_tile* __restrict__ tiles, const int* __restrict__ counts,
                                                           const int* __restrict__ rowtab, qmm_xmx x, void* __restrict__ D, int N, int K128,
                                                           uint32_t nblocks, int vec) {
    extern __shared__ __align__(16) uint8_t smem[];
    const uint32_t ti = blockIdx.x / nblocks;
    if (ti >= (uint32_t)(counts[0] + counts[1])) return;
    const qmm_moe_tile t = tiles[ti];
    const int n0 = (int)(blockIdx.x - ti * nblocks) * kMoeCols;
    const uint8_t* We = t.expert < 0 ? (Wsh ? Wsh : W) : W + (size_t)t.expert * ebytes;
    for (int r = 0; r < t.ncols; r += kMoeRows) {
        const int n = min(t.ncols - r, kMoeRows);
        if (n <= 32) moe_rows<1, BF>(smem, We, x, rowtab, t.k0 + r, n, n0, D, N, K128, vec);
        else moe_rows<2, BF>(smem, We, x, rowtab, t.k0 + r, n, n0, D, N, K128, vec);
        __syncthreads();                                 // LDS is filled again
    }
}

bool misaligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }

// what every product checks of its operands
int check_operands(const void* W, qmm_xmx x, const void* y, int dtype, int N, int K) {
    if (!W || !x.q || !x.e || !y) return QMM_ERR_NULL;
    if (dtype != QMM_F32 && dtype != QMM_BF16) return QMM_ERR_FORMAT;
    if (N <= 0 || K <= 0 || K > kMxMaxK) return QMM_ERR_SHAPE;
    if (misaligned(W, 16) || misaligned(x.q, 16) || misaligned(x.e, 4) || misaligned(y, dtype == QMM_BF16 ? 2 : 4)) return QMM_ERR_ARG;
    return QMM_OK;
}
// whether four outputs of a row are one aligned store, and whether 16 bytes of them are
int vec_out(const void* y, int dtype, int N) { return N % 4 == 0 && !misaligned(y, dtype == QMM_BF16 ? 8 : 16); }
int vec16_out(const void* y, int dtype, int N) { return N % (dtype == QMM_BF16 ? 8 : 4) == 0 && !misaligned(y, 16); }

struct GemmCall { const uint8_t* W; qmm_xmx x; void* D; int dtype, M, N, K128; hipStream_t s; };

template <class T, class F>
int launch_tiles(const GemmCall& c, F f) {
    const int64_t mt = ((int64_t)c.M + T::kRows - 1) / T::kRows, nt = ((int64_t)c.N + T::kCols - 1) / T::kCols;
    if (mt * nt > 0x7fffffff) return QMM_ERR_SHAPE;
    f(dim3((unsigned)(mt * nt)), (int)mt, vec16_out(c.D, c.dtype, c.N));
    QMM_LAUNCH_CHECK();
    return QMM_OK;
}
template <int MF, int NF, int D, int PER>
int launch_reg(const GemmCall& c) {
    using T = MxReg<MF, NF>;
    static_assert(T::kLds * PER <= 160 * 1024, "LDS of a CU");
    return launch_tiles<T>(c, [&](dim3 grid, int mt, int vec) {
        if (c.dtype == QMM_BF16)
            hipLaunchKernelGGL((k_gemm_mxfp4_reg<MF, NF, D, PER, true>), grid, dim3(256), T::kLds, c.s, c.W, c.x, c.D, c.M, c.N, c.K128, mt, vec);
        else
            hipLaunchKernelGGL((k_gemm_mxfp4_reg<MF, NF, D, PER, false>), grid, dim3(256), T::kLds, c.s, c.W, c.x, c.D, c.M, c.N, c.K128, mt, vec);
    });
}
template <int MF, int NF, int NS>
int launch_dma(const GemmCall& c) {
    using T = MxDma<MF, NF, NS>;
    static_assert(T::kLds <= 160 * 1024, "LDS of a CU");
    return launch_tiles<T>(c, [&](dim3 grid, int mt, int vec) {
        if (c.dtype == QMM_BF16)
            hipLaunchKernelGGL((k_gemm_mxfp4_dma<MF, NF, NS, true>), grid, dim3(512), T::kLds, c.s, c.W, c.x, c.D, c.M, c.N, c.K128, mt, vec);
        else
            hipLaunchKernelGGL((k_gemm_mxfp4_dma<MF, NF, NS, false>), grid, dim3(512), T::kLds, c.s, c.W, c.x, c.D, c.M, c.N, c.K128, mt, vec);
    });
}

// The tiles, and what a GEMM takes on each, in microseconds: a + steps (b + c (rounds - 1) + d load), rounds =
// ceil(tiles / 256 CUs), load = tiles / 256.  Fitted to 108 shapes (M 65 .. 4096, N 512 .. 17408, K 2048, 5120, 17408; mean
// error 2 to 10 %); the tile that it names takes 0.4 % more than the best of the seven on (geometric) average, 10 % at
// most.  Fewer tiles cost more: without the two DMA tiles 1.6 % (22 % at 4096 x 17408 x 2048), without 96 x 128 and 64 x 256 1 %
// (23 % at 512 x 5120 x 5120).
struct MxTileCost { int rows, cols; float a, b, c, d; int (*launch)(const GemmCall&); };
const MxTileCost kMxTiles[] = {
    {192, 384, 7.42f, 0.736f, 1.116f, 0.254f, launch_dma<3, 3, 3>}, {192, 256, 6.49f, 0.572f, 0.850f, 0.192f, launch_dma<3, 2, 4>},
    {128, 256, 5.48f, 0.415f, 0.558f, 0.185f, launch_reg<4, 2, 4, 1>}, {96, 128, 4.11f, 0.225f, 0.245f, 0.065f, launch_reg<3, 1, 8, 2>},
    {64, 256, 3.64f, 0.289f, 0.265f, 0.126f, launch_reg<2, 2, 4, 2>}, {64, 128, 4.00f, 0.180f, 0.208f, 0.051f, launch_reg<2, 1, 8, 2>},
    {32, 128, 4.22f, 0.129f, 0.134f, 0.028f, launch_reg<1, 1, 8, 2>},
};

const MxTileCost& pick_tile(int M, int N, int K128) {
    const MxTileCost* best = nullptr;
    float least = 0.f;
    for (const MxTileCost& t : kMxTiles) {
        const float tiles = (float)(((int64_t)M + t.rows - 1) / t.rows) * (float)(((int64_t)N + t.cols - 1) / t.cols);
        const float cost = t.a + (float)K128 * (t.b + t.c * (ceilf(tiles / 256.f) - 1.f) + t.d * tiles / 256.f);
        if (!best || cost < least) { best = &t; least = cost; }
    }
    return *best;
}

template <int MF>
int launch_gemv(const void* W, qmm_xmx x, void* y, int dtype, int ncol, int N, int K128, hipStream_t s) {
    const int S = gemv_waves(mx_groups(K128));
    const dim3 grid((unsigned)((N + 15) / 16)), block(64 * S);
    const size_t lds = (size_t)S * MF * 64 * sizeof(mx_v4f);
    if (dtype == QMM_BF16)
        hipLaunchKernelGGL((k_gemv_mxfp4<MF, true>), grid, block, lds, s, (const uint8_t*)W, x, y, N, K128, ncol, vec_out(y, dtype, N));
    else
        hipLaunchKernelGGL((k_gemv_mxfp4<MF, false>), grid, block, lds, s, (const uint8_t*)W, x, y, N, K128, ncol, vec_out(y, dtype, N));
    QMM_LAUNCH_CHECK();
    return QMM_OK;
}

}  // namespace
}  // namespace qmm

using namespace qmm;

extern "C" {

int qmm_gemv_mxfp4(const void* W, qmm_xmx x, void* y, int dtype, int ncol, int N, int K, void* stream) {
    const int st = check_operands(W, x, y, dtype, N, K);
    if (st != QMM_OK) return st;
    if (ncol < 0 || ncol > kGemvMaxRows) return QMM_ERR_SHAPE;
    if (ncol == 0) return QMM_OK;
    const int K128 = mx_steps(K);
    hipStream_t s = (hipStream_t)stream;
    if (ncol <= 16) return launch_gemv<1>(W, x, y, dtype, ncol, N, K128, s);
    if (ncol <= 32) return launch_gemv<2>(W, x, y, dtype, ncol, N, K128, s);
    return launch_gemv<4>(W, x, y, dtype, ncol, N, K128, s);
}

int qmm_gemv_moe_mxfp4(const void* W, const void* Wsh, size_t ebytes, const int* ids, qmm_xmx x, void* y, int dtype, int T, int nslot, int nexperts,
                       int N, int K, int xrow_te, void* stream) {
    const int st = check_operands(W, x, y, dtype, N, K);
    if (st != QMM_OK) return st;
    if (!ids) return QMM_ERR_NULL;
    if (T < 0 || T > kMoeGemvMaxT || nslot < 1 || nslot > kMoeMaxSlots || nexperts < 1) return QMM_ERR_SHAPE;
    if (ebytes % 16 != 0 || (nexperts > 1 && ebytes < qmm_mxfp4_weight_bytes(N, K)) || misaligned(Wsh, 16) || misaligned(ids, 4)) return QMM_ERR_ARG;
    if (T == 0) return QMM_OK;
    const int K128 = mx_steps(K), S = gemv_waves(mx_groups(K128));
    const dim3 grid((unsigned)((N + 15) / 16), (unsigned)(T * nslot)), block(64 * S);
    const size_t lds = (size_t)S * 64 * sizeof(mx_v4f);
    hipStream_t s = (hipStream_t)stream;
    if (dtype == QMM_BF16)
        hipLaunchKernelGGL(k_gemv_moe_mxfp4<true>, grid, block, lds, s, (const uint8_t*)W, (const uint8_t*)Wsh, ebytes, ids, x, y, T * nslot, nslot,
                           xrow_te, nexperts, N, K128, vec_out(y, dtype, N));
    else
        hipLaunchKernelGGL(k_gemv_moe_mxfp4<false>, grid, block, lds, s, (const uint8_t*)W, (const uint8_t*)Wsh, ebytes, ids, x, y, T * nslot, nslot,
                           xrow_te, nexperts, N, K128, vec_out(y, dtype, N));
    QMM_LAUNCH_CHECK();
    return QMM_OK;
}

int qmm_gemm_mxfp4(const void* W, qmm_xmx x, void* D, int dtype, int M, int N, int K, void* stream) {
    const int st = check_operands(W, x, D, dtype, N, K);
    if (st != QMM_OK) return st;
    if (M < 0) return QMM_ERR_SHAPE;
    if (M == 0) return QMM_OK;
    const int K128 = mx_steps(K);
    hipStream_t s = (hipStream_t)stream;
    return pick_tile(M, N, K128).launch(GemmCall{(const uint8_t*)W, x, D, dtype, M, N, K128, s});
}

int qmm_gemm_mxfp4_tile(int M, int N, int K) {
    if (M <= 0 || N <= 0 || K <= 0 || K > kMxMaxK) return QMM_ERR_SHAPE;
    return (int)(&pick_tile(M, N, mx_steps(K)) - kMxTiles);
}

int qmm_moe_gemm_mxfp4(const void* W, const void* Wsh, size_t ebytes, const qmm_moe_tile* tiles, const int* counts, int max_tiles, const int* rowtab,
                       qmm_xmx x, void* D, int dtype, int N, int K, void* stream) {
    const int st = check_operands(W, x, D, dtype, N, K);
    if (st != QMM_OK) return st;
    if (!tiles || !counts) return QMM_ERR_NULL;
    if (max_tiles < 0) return QMM_ERR_SHAPE;
    if (ebytes % 16 != 0 || misaligned(Wsh, 16) || misaligned(tiles, 4) || misaligned(counts, 4) || misaligned(rowtab, 4)) return QMM_ERR_ARG;
    if (max_tiles == 0) return QMM_OK;
    const uint32_t nblocks = ((uint32_t)N + kMoeCols - 1) / kMoeCols;
    if ((uint64_t)nblocks * max_tiles > 0x7fffffffu) return QMM_ERR_SHAPE;
    const int K128 = mx_steps(K);
    const dim3 grid(nblocks * (uint32_t)max_tiles);
    constexpr size_t lds = MxReg<kMoeRows / 32, kMoeNF>::kLds;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == QMM_BF16)
        hipLaunchKernelGGL(k_moe_gemm_mxfp4<true>, grid, dim3(256), lds, s, (const uint8_t*)W, (const uint8_t*)Wsh, ebytes, tiles, counts, rowtab, x, D, N,
                           K128, nblocks, vec16_out(D, dtype, N));
    else
        hipLaunchKernelGGL(k_moe_gemm_mxfp4<false>, grid, dim3(256), lds, s, (const uint8_t*)W, (const uint8_t*)Wsh, ebytes, tiles, counts, rowtab, x, D, N,
                           K128, nblocks, vec16_out(D, dtype, N));
    QMM_LAUNCH_CHECK();
    return QMM_OK;
}

}  // extern "C"
