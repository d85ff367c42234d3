// mx_gemm.hip -- products of MXFP4 activations and MXFP4 weights on the scaled matrix cores (layouts: mx.hpp):
//
//   qmm_gemv_mxfp4       y[m][n] = W[n] . x[m], m < 64: decode and draft verification
//   qmm_gemv_moe_mxfp4   the same for the routed experts of up to 16 tokens, by ids
//   qmm_gemm_mxfp4       any number of rows: prompts
//   qmm_moe_gemm_mxfp4   rows sorted by expert (qmm_moe_sort); _n with the sizes of its buffers
//
// v_mfma_scale_f32_32x32x64_f8f6f4 multiplies 32 weight rows by 32 activation rows over 64 values with their block
// scales and adds to f32 (16 x 16 over 128 reads twice the operand bytes per product: 5.4 against 6.4 PFLOP/s from
// registers).  The weight is the first operand, so a lane ends with runs of four successive outputs of one
// activation row.
//
// Order of sums.  GEMM: an output is one chain of instructions over K, whatever the tile, M or N.  GEMV: K's groups of
// four steps are cut into S contiguous runs, S chosen by K alone; each run is one chain and the S sums are added in
// order.  So an output's bits depend on its own rows and K, not on the call.
#include "mx_tile.hpp"

#include <algorithm>
#include <climits>
#include <cmath>

namespace qmm {
namespace {

// ------------------------------------------------------------------------------------------
// GEMV.  A workgroup is two strips (32 weight rows), its S waves the runs of K.  A wave reads its weights straight into
// the operand registers, by kilobytes, two steps (a pair) at a time, the next pair in flight while one is multiplied.
// The activation rows beside them come as whole 128-byte lines (a pair of a row, eight lanes) and turn into operands in
// LDS that is the wave's own: loaded in operand order, 16 bytes of 32 rows at a time, four loads touch each line, and the
// vector cache holds every load up whose line is still on its way (24 rows x 5120 x 17408 took twice the time).
// More than 32 rows are passes of 32, side by side: the weights of the second mostly come from caches (both fragments in one
// pass took 80 us at 64 rows x 17408 x 5120, for a cause not found).  With weights from memory / from the last-level cache: 1 row x
// 17408 x 5120 13.5 / 10.4 us (3.5 / 4.6 TB/s), 33 rows 22 / 20, 64 rows 25 / 22; 24 rows x 5120 x 17408 18 / 12.5, whose 160
// workgroups leave CUs idle.
constexpr int kGemvMaxWaves = 8, kGemvMaxRows = 64;

// S for G groups: one wave a group up to 8, else the count of 4 .. 8 that leaves the least imbalance
int gemv_waves(int G) {
    if (G <= kGemvMaxWaves) return G;
    int best = 4;
    for (int s = 5; s <= kGemvMaxWaves; ++s)
        if ((G + s - 1) / s * s <= (G + best - 1) / best * best) best = s;
    return best;
}

// LDS of one wave: a pair of 32 rows, and a group's scales of them (16 bytes a row)
constexpr int kGemvWaveLds = 32 * (128 + 16);

// LDS accesses of a wave before it stay before those after it (no instruction: a wave's LDS accesses are carried out in order,
// but the compiler may swap a lane's own read and write of different addresses, which are another lane's same ones)
__device__ __forceinline__ void wave_lds_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local"); }

// this wave's run of K: weight rows of `strip` and the next strip (sb bytes on, or 0 where there is none); row(r):
// the activation row of tile row r, of which n are real.  No branch lies around a load (the compiler would wait for
// every load in flight where the paths meet): the last group is a body of its own.
// QN: eights of activation rows that are loaded (1, 2 or 4)
template <int QN, class Row>
__device__ __forceinline__ void gemv_run(uint8_t* lds, const uint8_t* strip, uint32_t sb, qmm_xmx x, int n, Row row, int K128, int S, int wave,
                                         mx_v16f (&acc)[1][1]) {
    const int lane = threadIdx.x & 63, half = lane >> 5, G = mx_groups(K128), last = K128 - 1;
    const int g0 = wave * G / S, g1 = (wave + 1) * G / S;
    const uint8_t* wp = strip + ((lane & 16) ? sb : 0u);
    const uint32_t slot = (uint32_t)(half * 16 + (lane & 15));
    const uint8_t* qp[QN];                               // chunk lane % 8 of rows lane / 8 + 8 i
    const int cj = lane & 7;
#pragma unroll
    for (int i = 0; i < QN; ++i) qp[i] = x.q + (size_t)row(min(8 * i + (lane >> 3), n - 1)) * K128 * 64 + (cj & 3) * 16;
    const int fr = lane & 31, sw = a_swz(fr);            // the tile row of this lane's operand, whose scales it brings
    const uint8_t* ep = x.e + (size_t)row(min(fr, n - 1)) * K128 * 4;
    struct Pair { uint4 w[2][2], a[QN]; };
    struct Scales { uint32_t w[2], a[4]; };
    auto load = [&](Pair& r, int p) {                    // a step past the end re-reads the last one, unused
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int h = 0; h < 2; ++h) r.w[s][h] = ld16(wp + (uint32_t)min(2 * p + s, last) * 1024u + slot * 16u + h * 512u);
        const uint32_t off = (uint32_t)min(2 * p + (cj >> 2), last) * 64u;
#pragma unroll
        for (int i = 0; i < QN; ++i) r.a[i] = ld16(qp[i] + off);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto load_s = [&](Scales& r, int g) {
        const uint32_t sc = (uint32_t)K128 * 1024u + (uint32_t)g * 256u + slot * 4u;
        r.w[0] = *(const uint32_t*)(wp + sc);
        r.w[1] = *(const uint32_t*)(wp + sc + 128u);
#pragma unroll
        for (int s = 0; s < 4; ++s) r.a[s] = *(const uint32_t*)(ep + 4u * (uint32_t)min(4 * g + s, last));
    };
    const uint8_t* d = lds + fr * 128;
    uint8_t* es = lds + 32 * 128 + fr * 16;
    // the products of pair P of a group, `steps` (1 or 2) of them
    auto mul = [&](const Pair& r, const Scales& sc, auto pc, int steps) {
        constexpr int P = decltype(pc)::value;
#pragma unroll
        for (int i = 0; i < QN; ++i) {
            const int q = 8 * i + (lane >> 3);
            *(uint4*)(lds + q * 128 + ((cj ^ a_swz(q)) << 4)) = r.a[i];
        }
        wave_lds_fence();                                // other lanes read what this one wrote
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            if (s == steps) break;
            const uint4 a0 = *(const uint4*)(d + (((4 * s + half) ^ sw) << 4)), a1 = *(const uint4*)(d + (((4 * s + 2 + half) ^ sw) << 4));
            const uint32_t sa = *(const uint32_t*)(es + 4 * (2 * P + s)) >> (8 * half);
            if (s == 0) {
                acc[0][0] = mx_mfma32<2 * P, 0>(r.w[0][0], a0, acc[0][0], sc.w[0], sa);
                acc[0][0] = mx_mfma32<2 * P, 2>(r.w[0][1], a1, acc[0][0], sc.w[1], sa);
            } else {
                acc[0][0] = mx_mfma32<2 * P + 1, 0>(r.w[1][0], a0, acc[0][0], sc.w[0], sa);
                acc[0][0] = mx_mfma32<2 * P + 1, 2>(r.w[1][1], a1, acc[0][0], sc.w[1], sa);
            }
        }
        wave_lds_fence();                                // the reads come before the next pair's writes
        pin<false>(acc[0][0]);
        __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[0][0][e] = 0.f;
    if (g0 < g1) {
        Pair r0, r1;
        Scales sc;
        load_s(sc, g0);
        load(r0, 2 * g0);
        load(r1, 2 * g0 + 1);
        for (int g = g0; g < g1 - 1; ++g) {
            *(uint4*)es = make_uint4(sc.a[0], sc.a[1], sc.a[2], sc.a[3]);
            const Scales now = sc;
            mul(r0, now, std::integral_constant<int, 0>{}, 2);
            load_s(sc, g + 1);
            load(r0, 2 * g + 2);
            mul(r1, now, std::integral_constant<int, 1>{}, 2);
            load(r1, 2 * g + 3);
        }
        const int left = K128 - 4 * (g1 - 1);            // steps of the last group (beyond 4: whole)
        *(uint4*)es = make_uint4(sc.a[0], sc.a[1], sc.a[2], sc.a[3]);
        mul(r0, sc, std::integral_constant<int, 0>{}, min(left, 2));
        if (left > 2) mul(r1, sc, std::integral_constant<int, 1>{}, min(left - 2, 2));
    }
    settle<false>(acc);
}

// The S runs' sums, added in order: item i = 64 e + lane of the tile, four outputs each (weight rows 8 e ..)
__device__ __forceinline__ void gemv_reduce(mx_v4f* red, const mx_v16f (&acc)[1][1], int wave) {
    __syncthreads();                                     // the same LDS held the waves' operands
    const mx_v16f& a = acc[0][0];
#pragma unroll
    for (int e = 0; e < 4; ++e) red[(wave * 4 + e) * 64 + (threadIdx.x & 63)] = mx_v4f{a[4 * e], a[4 * e + 1], a[4 * e + 2], a[4 * e + 3]};
    __syncthreads();
}
__device__ __forceinline__ mx_v4f gemv_sum(const mx_v4f* red, int i, int S) {
    mx_v4f v = red[i];
    for (int w = 1; w < S; ++w) v += red[w * 256 + i];
    return v;
}

// Workgroup (two strips, pass): pass p takes the rows 8 QN p ..
template <int QN, bool BF>
__global__ void __launch_bounds__(64 * kGemvMaxWaves) k_gemv_mxfp4(const uint8_t* __restrict__ W, qmm_xmx x, void* __restrict__ y, int N, int K128,
                                                                   int ncol, int vec) {
    extern __shared__ __align__(16) uint8_t smem[];
    mx_v4f* red = (mx_v4f*)smem;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), S = blockDim.x >> 6;
    const int n0 = (int)blockIdx.x * 32, m0 = (int)blockIdx.y * 8 * QN, m1 = min(m0 + 8 * QN, ncol);
    const uint32_t sb = mx_strip_bytes(K128);
    mx_v16f acc[1][1];
    gemv_run<QN>(smem + wave * kGemvWaveLds, W + (size_t)blockIdx.x * 2 * sb, n0 + 16 < N ? sb : 0u, x, m1 - m0, [&](int r) { return m0 + r; }, K128, S,
                 wave, acc);
    gemv_reduce(red, acc, wave);
    for (int i = threadIdx.x; i < 256; i += blockDim.x) {
        const int m = m0 + (i & 31), n = n0 + 8 * (i >> 6) + 4 * ((i >> 5) & 1);
        if (m < m1 && n < N) mx_store4<BF>(y, (size_t)m * N + n, gemv_sum(red, i, S), N - n, vec);
    }
}

// Experts by ids: workgroup (two strips, slot).  The first slot of an expert computes all slots that hold it, 8 QN at
// a time (a token lists an expert once, so T tokens make one pass), the others leave: an expert is read once.
constexpr int kMoeGemvMaxT = 16, kMoeGemvMaxSlots = kMoeGemvMaxT * kMoeMaxSlots;

template <int QN, bool BF>
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
    const int n0 = (int)blockIdx.x * 32;
    const uint32_t sb = mx_strip_bytes(K128);
    const uint8_t* strip = (id < 0 ? Wsh : W + (size_t)id * ebytes) + (size_t)blockIdx.x * 2 * sb;
    for (int c0 = 0; c0 < n; c0 += 8 * QN) {
        mx_v16f acc[1][1];
        gemv_run<QN>(smem + wave * kGemvWaveLds, strip, n0 + 16 < N ? sb : 0u, x, min(n - c0, 8 * QN), [&](int r) {
            const int slot = cols[c0 + r];
            return xrow_te ? slot : slot / per_token;
        }, K128, S, wave, acc);
        gemv_reduce(red, acc, wave);
        for (int i = threadIdx.x; i < 256; i += blockDim.x) {
            const int c = c0 + (i & 31), nn = n0 + 8 * (i >> 6) + 4 * ((i >> 5) & 1);
            if ((i & 31) < 8 * QN && c < n && nn < N) mx_store4<BF>(y, (size_t)cols[c] * N + nn, gemv_sum(red, i, S), N - nn, vec);
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

// Grouped: workgroup (tile of one expert's rows, block of 128 outputs); a tile's rows 128 at a time, with as
// many 32-row fragments as they need.  512 experts of 1024 x 2048, 10 a token and a shared one: 512 tokens 109 us, 2048
// 127, 8192 248; 64 rows at a time 335 at 8192 (weights are read again).  The 571 MB of weights take 110 at a large
// copy's rate, and bound it up to 2048 tokens; beyond, the steps of the tiles do.  Weights three steps ahead: seven take
// 5 % more at 2048, a third workgroup on a CU (of 168 registers a wave) 12 %.
constexpr int kMoeNF = 1, kMoeD = 4, kMoeCols = 128 * kMoeNF, kMoeRows = 128;

//
// The tiles and the table come from the device, where no host check sees them: an expert or a row beyond what the caller says
// the buffers hold is taken as the last one, and rows of D beyond its end are left out.
struct MoeBounds { int experts, rows, xrows; };

template <int MF, bool BF>
__device__ __forceinline__ void moe_rows(uint8_t* smem, const uint8_t* We, qmm_xmx x, const int* rowtab, int xrows, int k0, int n, int n0, void* D, int N,
                                         int K128, int vec) {
    mx_v16f acc[kMoeNF][MF];
    mx_tile_reg<MF, kMoeNF, kMoeD, false>(smem, We, x, n0 / 16, (N + 15) / 16, K128, [&](int r) {
        const int k = k0 + min(r, n - 1);
        return rowtab ? rowtab[k] : k;
    }, acc, [&](int row) { return min(max(row, 0), xrows - 1); });
    mx_store<MF, kMoeNF, BF>(smem, acc, D, n0 + 32 * kMoeNF * (int)(threadIdx.x >> 6), N, vec, [&](int r) { return r < n ? (int64_t)(k0 + r) : -1; });
}

template <bool BF>
__global__ void __launch_bounds__(256, 2) k_moe_gemm_mxfp4(const uint8_t* __restrict__ W, const uint8_t* __restrict__ Wsh, size_t ebytes,
                                                           const qmm_moe_tile* __restrict__ tiles, const int* __restrict__ counts,
                                                           const int* __restrict__ rowtab, qmm_xmx x, void* __restrict__ D, int N, int K128,
                                                           uint32_t nblocks, int vec, MoeBounds b) {
    extern __shared__ __align__(16) uint8_t smem[];
    const uint32_t ti = blockIdx.x / nblocks;
    if (ti >= (uint32_t)(counts[0] + counts[1])) return;
    const qmm_moe_tile t = tiles[ti];
    const int n0 = (int)(blockIdx.x - ti * nblocks) * kMoeCols;
    const uint8_t* We = t.expert < 0 ? (Wsh ? Wsh : W) : W + (size_t)min(t.expert, b.experts - 1) * ebytes;
    const int rows = t.k0 < 0 ? 0 : min(t.ncols, b.rows - t.k0);
    for (int r = 0; r < rows; r += kMoeRows) {
        const int n = min(rows - r, kMoeRows);
        if (n <= 32) moe_rows<1, BF>(smem, We, x, rowtab, b.xrows, t.k0 + r, n, n0, D, N, K128, vec);
        else if (n <= 64) moe_rows<2, BF>(smem, We, x, rowtab, b.xrows, t.k0 + r, n, n0, D, N, K128, vec);
        else if (n <= 96) moe_rows<3, BF>(smem, We, x, rowtab, b.xrows, t.k0 + r, n, n0, D, N, K128, vec);
        else moe_rows<4, BF>(smem, We, x, rowtab, b.xrows, t.k0 + r, n, n0, D, N, K128, vec);
        __syncthreads();                                 // LDS is filled again
    }
}

bool misaligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }

// what every product checks of its operands (rows: 0 if it has none, and then needs no buffers of them)
int check_operands(const void* W, qmm_xmx x, const void* y, int dtype, int rows, int N, int K) {
    if (!W || (rows != 0 && (!x.q || !x.e || !y))) return QMM_ERR_NULL;
    if (dtype != QMM_F32 && dtype != QMM_BF16) return QMM_ERR_FORMAT;
    if (N <= 0 || N > kMxMaxRows || K <= 0 || K > kMxMaxK) return QMM_ERR_SHAPE;
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
    if (!grid_fits((uint64_t)(mt * nt), T::kThreads)) return QMM_ERR_SHAPE;
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
// ceil(tiles / 256 CUs), load = tiles / 256.  Fitted to calls one by one (4 to 18 % off the times in a replayed
// graph).  Over 108 shapes (M 65 .. 4096, N 512 .. 17408, K 2048, 5120, 17408) the tile that they name takes 0.3 % more
// than the best of the eight on (geometric) average, 11 % at most; without one of the first seven 0.9 to 5.7 % (14 to
// 37 % at most), without 192 x 128 0.6 % (1024 x 5120 x 5120 takes 26 us instead of 22).
struct MxTileCost { int rows, cols; float a, b, c, d; int (*launch)(const GemmCall&); };
const MxTileCost kMxTiles[] = {
    {192, 384, 7.42f, 0.736f, 1.116f, 0.254f, launch_dma<3, 3, 3>}, {192, 256, 6.49f, 0.572f, 0.850f, 0.192f, launch_dma<3, 2, 4>},
    {128, 256, 5.48f, 0.415f, 0.558f, 0.185f, launch_reg<4, 2, 4, 1>}, {96, 128, 4.11f, 0.225f, 0.245f, 0.065f, launch_reg<3, 1, 4, 2>},
    {64, 256, 3.64f, 0.289f, 0.265f, 0.126f, launch_reg<2, 2, 4, 2>}, {64, 128, 4.00f, 0.180f, 0.208f, 0.051f, launch_reg<2, 1, 4, 2>},
    {32, 128, 4.22f, 0.129f, 0.134f, 0.028f, launch_reg<1, 1, 8, 2>}, {192, 128, 5.10f, 0.339f, 0.433f, 0.201f, launch_reg<6, 1, 4, 1>},
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

template <int QN>
int launch_gemv(const void* W, qmm_xmx x, void* y, int dtype, int ncol, int N, int K128, hipStream_t s) {
    const int S = gemv_waves(mx_groups(K128));
    const dim3 grid((unsigned)((N + 31) / 32), (unsigned)((ncol + 8 * QN - 1) / (8 * QN))), block(64 * S);
    if (!grid_fits(grid.x, block.x)) return QMM_ERR_SHAPE;
    const size_t lds = (size_t)S * std::max<size_t>(256 * sizeof(mx_v4f), kGemvWaveLds);
    if (dtype == QMM_BF16)
        hipLaunchKernelGGL((k_gemv_mxfp4<QN, true>), grid, block, lds, s, (const uint8_t*)W, x, y, N, K128, ncol, vec_out(y, dtype, N));
    else
        hipLaunchKernelGGL((k_gemv_mxfp4<QN, false>), grid, block, lds, s, (const uint8_t*)W, x, y, N, K128, ncol, vec_out(y, dtype, N));
    QMM_LAUNCH_CHECK();
    return QMM_OK;
}

template <int QN>
int launch_gemv_moe(const void* W, const void* Wsh, size_t ebytes, const int* ids, qmm_xmx x, void* y, int dtype, int T, int nslot, int nexperts, int N,
                    int K128, int xrow_te, hipStream_t s) {
    const int S = gemv_waves(mx_groups(K128));
    const dim3 grid((unsigned)((N + 31) / 32), (unsigned)(T * nslot)), block(64 * S);
    if (!grid_fits(grid.x, block.x)) return QMM_ERR_SHAPE;
    const size_t lds = (size_t)S * std::max<size_t>(256 * sizeof(mx_v4f), kGemvWaveLds);
    if (dtype == QMM_BF16)
        hipLaunchKernelGGL((k_gemv_moe_mxfp4<QN, true>), grid, block, lds, s, (const uint8_t*)W, (const uint8_t*)Wsh, ebytes, ids, x, y, T * nslot, nslot,
                           xrow_te, nexperts, N, K128, vec_out(y, dtype, N));
    else
        hipLaunchKernelGGL((k_gemv_moe_mxfp4<QN, false>), grid, block, lds, s, (const uint8_t*)W, (const uint8_t*)Wsh, ebytes, ids, x, y, T * nslot, nslot,
                           xrow_te, nexperts, N, K128, vec_out(y, dtype, N));
    QMM_LAUNCH_CHECK();
    return QMM_OK;
}

int launch_moe_gemm(const void* W, const void* Wsh, size_t ebytes, const qmm_moe_tile* tiles, const int* counts, int max_tiles, const int* rowtab,
                    qmm_xmx x, void* D, int dtype, int N, int K, MoeBounds b, hipStream_t s) {
    if (ebytes % 16 != 0 || misaligned(Wsh, 16) || misaligned(tiles, 4) || misaligned(counts, 4) || misaligned(rowtab, 4)) return QMM_ERR_ARG;
    if (max_tiles == 0 || b.rows == 0) return QMM_OK;
    const uint32_t nblocks = ((uint32_t)N + kMoeCols - 1) / kMoeCols;
    if (!grid_fits((uint64_t)nblocks * max_tiles, 256)) return QMM_ERR_SHAPE;
    const int K128 = mx_steps(K);
    const dim3 grid(nblocks * (uint32_t)max_tiles);
    constexpr size_t lds = MxReg<kMoeRows / 32, kMoeNF>::kLds;
    if (dtype == QMM_BF16)
        hipLaunchKernelGGL(k_moe_gemm_mxfp4<true>, grid, dim3(256), lds, s, (const uint8_t*)W, (const uint8_t*)Wsh, ebytes, tiles, counts, rowtab, x, D, N,
                           K128, nblocks, vec16_out(D, dtype, N), b);
    else
        hipLaunchKernelGGL(k_moe_gemm_mxfp4<false>, grid, dim3(256), lds, s, (const uint8_t*)W, (const uint8_t*)Wsh, ebytes, tiles, counts, rowtab, x, D, N,
                           K128, nblocks, vec16_out(D, dtype, N), b);
    QMM_LAUNCH_CHECK();
    return QMM_OK;
}

}  // namespace
}  // namespace qmm

using namespace qmm;

extern "C" {

int qmm_gemv_mxfp4(const void* W, qmm_xmx x, void* y, int dtype, int ncol, int N, int K, void* stream) {
    const int st = check_operands(W, x, y, dtype, ncol, N, K);
    if (st != QMM_OK) return st;
    if (ncol < 0 || ncol > kGemvMaxRows) return QMM_ERR_SHAPE;
    if (ncol == 0) return QMM_OK;
    const int K128 = mx_steps(K);
    hipStream_t s = (hipStream_t)stream;
    if (ncol <= 8) return launch_gemv<1>(W, x, y, dtype, ncol, N, K128, s);
    if (ncol <= 16) return launch_gemv<2>(W, x, y, dtype, ncol, N, K128, s);
    return launch_gemv<4>(W, x, y, dtype, ncol, N, K128, s);
}

int qmm_gemv_moe_mxfp4(const void* W, const void* Wsh, size_t ebytes, const int* ids, qmm_xmx x, void* y, int dtype, int T, int nslot, int nexperts,
                       int N, int K, int xrow_te, void* stream) {
    const int st = check_operands(W, x, y, dtype, T, N, K);
    if (st != QMM_OK) return st;
    if (T != 0 && !ids) return QMM_ERR_NULL;
    if (T < 0 || T > kMoeGemvMaxT || nslot < 1 || nslot > kMoeMaxSlots || nexperts < 1) return QMM_ERR_SHAPE;
    if (ebytes % 16 != 0 || (nexperts > 1 && ebytes < qmm_mxfp4_weight_bytes(N, K)) || misaligned(Wsh, 16) || misaligned(ids, 4)) return QMM_ERR_ARG;
    if (T == 0) return QMM_OK;
    if (T <= 8) return launch_gemv_moe<1>(W, Wsh, ebytes, ids, x, y, dtype, T, nslot, nexperts, N, mx_steps(K), xrow_te, (hipStream_t)stream);
    return launch_gemv_moe<2>(W, Wsh, ebytes, ids, x, y, dtype, T, nslot, nexperts, N, mx_steps(K), xrow_te, (hipStream_t)stream);
}

int qmm_gemm_mxfp4(const void* W, qmm_xmx x, void* D, int dtype, int M, int N, int K, void* stream) {
    const int st = check_operands(W, x, D, dtype, M, N, K);
    if (st != QMM_OK) return st;
    if (M < 0 || M > kMxMaxRows) return QMM_ERR_SHAPE;
    if (M == 0) return QMM_OK;
    const int K128 = mx_steps(K);
    hipStream_t s = (hipStream_t)stream;
    return pick_tile(M, N, K128).launch(GemmCall{(const uint8_t*)W, x, D, dtype, M, N, K128, s});
}

int qmm_gemm_mxfp4_tile(int M, int N, int K) {
    if (M <= 0 || M > kMxMaxRows || N <= 0 || N > kMxMaxRows || K <= 0 || K > kMxMaxK) return QMM_ERR_SHAPE;
    return (int)(&pick_tile(M, N, mx_steps(K)) - kMxTiles);
}

int qmm_moe_gemm_mxfp4_n(const void* W, const void* Wsh, size_t ebytes, int nexperts, const qmm_moe_tile* tiles, const int* counts, int max_tiles,
                         const int* rowtab, int rows, qmm_xmx x, int xrows, void* D, int dtype, int N, int K, void* stream) {
    const int st = check_operands(W, x, D, dtype, rows, N, K);
    if (st != QMM_OK) return st;
    if (!tiles || !counts) return QMM_ERR_NULL;
    if (max_tiles < 0 || nexperts < 1 || rows < 0 || xrows < (rowtab ? (rows > 0) : rows)) return QMM_ERR_SHAPE;
    if (nexperts > 1 && ebytes < qmm_mxfp4_weight_bytes(N, K)) return QMM_ERR_ARG;
    return launch_moe_gemm(W, Wsh, ebytes, tiles, counts, max_tiles, rowtab, x, D, dtype, N, K, MoeBounds{nexperts, rows, xrows}, (hipStream_t)stream);
}

int qmm_moe_gemm_mxfp4(const void* W, const void* Wsh, size_t ebytes, const qmm_moe_tile* tiles, const int* counts, int max_tiles, const int* rowtab,
                       qmm_xmx x, void* D, int dtype, int N, int K, void* stream) {
    const int st = check_operands(W, x, D, dtype, 1, N, K);
    if (st != QMM_OK) return st;
    if (!tiles || !counts) return QMM_ERR_NULL;
    if (max_tiles < 0) return QMM_ERR_SHAPE;
    return launch_moe_gemm(W, Wsh, ebytes, tiles, counts, max_tiles, rowtab, x, D, dtype, N, K, MoeBounds{INT_MAX, INT_MAX, INT_MAX}, (hipStream_t)stream);
}

}  // extern "C"
