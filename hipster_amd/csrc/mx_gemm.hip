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
#include "mx.hpp"

#include <algorithm>
#include <type_traits>

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
// GEMM tile, on v_mfma_scale_f32_32x32x64_f8f6f4.  WM x WN waves; a wave owns 32 MF activation rows and 32 NF
// weight rows.  Both operands come by DMA (global_load_lds):
//   - activations two steps (a pair, 128 bytes of a row: whole cache lines) at a time into NA buffers, 16-byte
//     chunk c of a row at chunk c ^ swz(row).  Half lines, one step at a time, cost the vector cache a stall for
//     every second half (the line is still on its way): half of all cycles, 155 instead of XX us below;
//   - weights step by step into a ring of NS, a strip's kilobyte as it is in memory;
//   - block scales by groups of four steps, 16 bytes a row, into two buffers.
// The operand reads (16 lanes: 16 rows, one chunk) are free of bank conflicts.  A step k is: wait until the own
// DMAs that it reads have landed, barrier, start those NS - 1 steps (pairs: NA - 1 pairs) ahead, whose buffers were
// read before that barrier, multiply.
//
// Eight waves run as two halves (the rows' halves, one wave of each on a SIMD), half a step apart: while one half reads
// its operands from LDS and issues its DMAs, the other multiplies, and a barrier ends each phase.
__device__ __forceinline__ int a_swz(int row) { return ((row >> 1) & 7) ^ ((row & 1) << 2); }

template <int MF, int NF, int WM, int WN, int NS, int NA>
struct MxTile {
    static constexpr int kWaves = WM * WN, kRows = 32 * MF * WM, kCols = 32 * NF * WN;
    static constexpr int per(int pieces) { return (pieces + kWaves - 1) / kWaves; }
    // DMAs (1 KB each): of a pair's activations, of a step's weights, of a group's scales; and per wave
    static constexpr int kAPieces = kRows / 8, kWPieces = kCols / 16, kRowSc = (kRows + 63) / 64, kScPieces = kRowSc + (kCols + 63) / 64;
    static constexpr int PA = per(kAPieces), PW = per(kWPieces), PS = per(kScPieces);
    static constexpr int kABytes = kAPieces * 1024, kWBytes = kWPieces * 1024, kScBytes = kScPieces * 1024;
    static constexpr int kWAt = NA * kABytes, kScAt = kWAt + NS * kWBytes, kLoopLds = kScAt + 2 * kScBytes;
    static constexpr int kStoreLds = kWaves * 32 * (128 * NF + 16), kLds = kLoopLds > kStoreLds ? kLoopLds : kStoreLds;
    // eight waves, two on each SIMD: they work half a step apart
    static constexpr bool kTwo = kWaves == 8;
    static_assert(!kTwo || WM == 2, "the two halves are the waves 0 .. 3 and 4 .. 7");
    // what a wave issues in step j (mod 4): scales of the next group, a pair, a step of weights, in this order
    static constexpr int issued(int j) { return PW + ((j & 1) == 0 ? PA : 0) + ((j & 3) == 0 ? PS : 0); }
    static constexpr int issued(int from, int to) { return from > to ? 0 : issued(from) + issued(from + 1, to); }
    // DMAs younger than those that step k (mod 4, plus a multiple of 4) reads
    static constexpr int younger(int k) {
        const int w = issued(k - NS + 2, k - 1), a = PW + issued(k - 2 * (NA - 1) + 1, k - 1);
        return (k & 1) == 0 && a < w ? a : w;
    }
    static_assert(NS >= 3 && NS <= 4 && NA >= 2 && NA <= 3, "the waits below hold for these");
};

// s_waitcnt vmcnt(n)
template <int N>
__device__ __forceinline__ void vm_wait() {
    static_assert(N >= 0 && N < 64, "vmcnt has six bits");
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}

// the value exists here, in registers (no instruction)
__device__ __forceinline__ void pin(uint32_t& v) { asm volatile("" : "+v"(v)); }
__device__ __forceinline__ void pin(mx_v16f& v) { asm volatile("" : "+v"(v)); }
__device__ __forceinline__ void pin(uint4& a, uint4& b) {
    asm volatile("" : "+v"(a.x), "+v"(a.y), "+v"(a.z), "+v"(a.w), "+v"(b.x), "+v"(b.y), "+v"(b.z), "+v"(b.w));
}
template <int I, int N, class F>
__device__ __forceinline__ void static_for(F f) {
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        static_for<I + 1, N>(f);
    }
}

// rows(r): the activation row of tile row r.  acc[f][j]: weight rows 32 f.., activation rows 32 j.. of this wave
template <int MF, int NF, int WM, int WN, int NS, int NA, class Rows>
__device__ __forceinline__ void mx_tile(uint8_t* smem, const uint8_t* W, qmm_xmx x, int strip0, int nstrips, int K128, Rows rows, mx_v16f (&acc)[NF][MF]) {
    using T = MxTile<MF, NF, WM, WN, NS, NA>;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wn = wave % WN, wm = wave / WN, half = lane >> 5;
    const uint32_t lds = lds_addr(smem);

    // this wave's pieces (where the waves do not divide them, the last one is fetched more than once): eight
    // activation rows, a strip, 64 rows' scales (16 bytes; the last group of a row starts at step K128 - 4, so that
    // it ends with the row) or four strips' scales (256 bytes)
    const uint8_t* ap[T::PA];
    uint32_t adst[T::PA];
    bool late[T::PA];                                    // the lane's chunk is of the pair's second step
#pragma unroll
    for (int i = 0; i < T::PA; ++i) {
        const int p = min(wave + i * T::kWaves, T::kAPieces - 1), r = 8 * p + (lane >> 3), c = (lane & 7) ^ a_swz(r);
        adst[i] = lds + (uint32_t)p * 1024u;
        ap[i] = x.q + (size_t)rows(r) * K128 * 64 + c * 16;
        late[i] = c >= 4;
    }
    const uint8_t* wp[T::PW];
    uint32_t wdst[T::PW];
#pragma unroll
    for (int i = 0; i < T::PW; ++i) {
        const int p = min(wave + i * T::kWaves, T::kWPieces - 1);
        wdst[i] = lds + T::kWAt + (uint32_t)p * 1024u;
        wp[i] = W + (size_t)min(strip0 + p, nstrips - 1) * mx_strip_bytes(K128) + lane * 16;
    }
    const uint8_t* sp[T::PS];
    uint32_t sdst[T::PS];
    bool srow[T::PS];
#pragma unroll
    for (int i = 0; i < T::PS; ++i) {
        const int p = min(wave + i * T::kWaves, T::kScPieces - 1);
        sdst[i] = lds + T::kScAt + (uint32_t)p * 1024u;
        srow[i] = p < T::kRowSc;
        if (srow[i]) sp[i] = x.e + (size_t)rows(min(64 * p + lane, T::kRows - 1)) * K128 * 4;
        else sp[i] = W + (size_t)min(strip0 + min(4 * (p - T::kRowSc) + (lane >> 4), T::kCols / 16 - 1), nstrips - 1) * mx_strip_bytes(K128) +
                     (uint32_t)K128 * 1024u + (lane & 15) * 16;
    }
    auto issue_a = [&](int i, int pair, int buf) {       // piece i of a pair
        const bool odd = 2 * pair + 1 >= K128;           // the pair's second step does not exist: the first again
        dma16(ap[i] - (odd && late[i] ? 64 : 0), adst[i] + buf * T::kABytes);
        ap[i] += 128;
    };
    auto issue_w = [&](int i, int buf) {
        dma16(wp[i], wdst[i] + buf * T::kWBytes);
        wp[i] += 1024;
    };
    auto issue_s = [&](int i, int g) {
        const uint32_t off = srow[i] ? (uint32_t)max(min(4 * g, K128 - 4), 0) * 4u : (uint32_t)g * 256u;
        if (!srow[i] || K128 >= 4) dma16(sp[i] + off, sdst[i] + (g & 1) * T::kScBytes);
    };
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int j = 0; j < MF; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[f][j][e] = 0.f;

    if (K128 < 4) {                                      // rows shorter than a 16-byte piece of scales
        for (int i = tid; i < T::kRows * K128; i += 64 * T::kWaves) {
            const int r = i / K128, s = i - r * K128;
            *(uint32_t*)(smem + T::kScAt + r * 16 + s * 4) = *(const uint32_t*)(x.e + ((size_t)rows(r) * K128 + s) * 4);
        }
    }
#pragma unroll
    for (int i = 0; i < T::PS; ++i) issue_s(i, 0);
#pragma unroll
    for (int p = 0; p < NA - 1; ++p)
        if (2 * p < K128)
#pragma unroll
            for (int i = 0; i < T::PA; ++i) issue_a(i, p, p);
#pragma unroll
    for (int k = 0; k < NS - 1; ++k)
        if (k < K128)
#pragma unroll
            for (int i = 0; i < T::PW; ++i) issue_w(i, k);

    const int r0 = wm * 32 * MF + (lane & 31), sw = a_swz(r0);                      // rows 32 apart: the same rotation
    const uint32_t a_at = (uint32_t)r0 * 128u;
    const uint32_t w_at = (uint32_t)(2 * wn * NF + ((lane >> 4) & 1)) * 1024u + (uint32_t)(half * 16 + (lane & 15)) * 16u;
    const uint32_t ws_at = (uint32_t)T::kScAt + T::kRowSc * 1024u + (uint32_t)(2 * wn * NF + ((lane >> 4) & 1)) * 256u +
                           (uint32_t)(half * 16 + (lane & 15)) * 4u;
    uint32_t ws[NF][2];
    int wbuf = 0, abuf = 0;
    // Everything that step k reads has landed in this wave's part.  S = k % 4 in the steady groups, where every DMA
    // exists and the wait is a constant; S = -1 for the first group and the last steps: at the start the pairs came
    // before the weights and near the end nothing new was issued, so only the weights of the steps after this one
    // may still be out (they are younger than everything that it reads).
    auto landed = [&](auto sc, int k) {
        constexpr int S = decltype(sc)::value;
        if constexpr (S >= 0) vm_wait<T::younger(S + 8)>();
        else if (K128 >= 4 && k + NS - 2 < K128) vm_wait<(NS - 2) * T::PW>();
        else if (K128 >= 4 && NS == 4 && k + 1 < K128) vm_wait<T::PW>();
        else vm_wait<0>();
    };
    using Next = std::integral_constant<int, -1>;
    auto step = [&](auto sc, auto nc, int k) {           // nc: S of the step after this one
        constexpr int S = decltype(sc)::value;
        constexpr bool kSteady = S >= 0;
        const int g = k >> 2;
        if constexpr (!T::kTwo) {
            landed(sc, k);
            lds_barrier();
        }
        const int an = abuf == 0 ? NA - 1 : abuf - 1, wn_ = wbuf == 0 ? NS - 1 : wbuf - 1;
        // the step's DMAs: part B of P
        auto issue = [&](auto bc, auto pc) {
            constexpr int B = decltype(bc)::value, P = decltype(pc)::value;
            constexpr int nS = S <= 0 ? T::PS : 0, nA = !kSteady || (S & 1) == 0 ? T::PA : 0, n = nS + nA + T::PW;
            constexpr int lo = B * n / P, hi = (B + 1) * n / P;
#pragma unroll
            for (int i = lo; i < hi; ++i) {
                if (i < nS) { if (kSteady || ((k & 3) == 0 && k + 4 < K128)) issue_s(i, g + 1); }
                else if (i < nS + nA) { if (kSteady || ((k & 1) == 0 && k + 2 * (NA - 1) < K128)) issue_a(i - nS, (k >> 1) + NA - 1, an); }
                else { if (kSteady || k + NS - 1 < K128) issue_w(i - nS - nA, wn_); }
            }
        };
        const uint8_t* sa_ = smem + abuf * T::kABytes + a_at;
        const uint8_t* sw_ = smem + T::kWAt + wbuf * T::kWBytes + w_at;
        const uint32_t so = (uint32_t)(g & 1) * T::kScBytes;
        if constexpr (S <= 0) {
#pragma unroll
            for (int f = 0; f < NF; ++f)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    ws[f][h] = *(const uint32_t*)(smem + ws_at + so + f * 512 + h * 128);
                    if constexpr (!kSteady) ws[f][h] >>= 8 * (k & 3);
                }
        }
        const int c0 = 4 * (k & 1) + half;               // the lane's first block
        const uint8_t* sa_row = smem + T::kScAt + so + r0 * 16 + 4 * (k - max(min(4 * g, K128 - 4), 0));
        uint4 w[NF][2], a[MF][2];
        uint32_t sa[MF];
        auto read_a = [&](int j) {
            a[j][0] = *(const uint4*)(sa_ + j * 4096 + ((c0 ^ sw) << 4));
            a[j][1] = *(const uint4*)(sa_ + j * 4096 + (((c0 + 2) ^ sw) << 4));
            // the step's four scale bytes, this lane's two in bytes 0 and 2
            sa[j] = *(const uint32_t*)(sa_row + j * 512) >> (8 * half);
        };
#pragma unroll
        for (int f = 0; f < NF; ++f)
#pragma unroll
            for (int h = 0; h < 2; ++h) w[f][h] = *(const uint4*)(sw_ + f * 2048 + h * 512);
        if constexpr (T::kTwo) {
#pragma unroll
            for (int j = 0; j < MF; ++j) read_a(j);
            issue(std::integral_constant<int, 0>{}, std::integral_constant<int, 1>{});
            // the compiler would move the reads and the products to where they suit it: they stay in their phases
#pragma unroll
            for (int f = 0; f < NF; ++f) pin(w[f][0], w[f][1]);
#pragma unroll
            for (int j = 0; j < MF; ++j) { pin(a[j][0], a[j][1]); pin(sa[j]); }
            if (wm != 0) landed(nc, k + 1);
            lds_barrier();
            __builtin_amdgcn_s_setprio(1);
        }
        static_for<0, MF>([&](auto jc) {
            constexpr int j = decltype(jc)::value;
            if constexpr (!T::kTwo) read_a(j);
#pragma unroll
            for (int f = 0; f < NF; ++f) acc[f][j] = mx_mfma32<kSteady ? S : 0, 0>(w[f][0], a[j][0], acc[f][j], ws[f][0], sa[j]);
            if constexpr (!T::kTwo) issue(std::integral_constant<int, 2 * j>{}, std::integral_constant<int, 2 * MF>{});
#pragma unroll
            for (int f = 0; f < NF; ++f) acc[f][j] = mx_mfma32<kSteady ? S : 0, 2>(w[f][1], a[j][1], acc[f][j], ws[f][1], sa[j]);
            if constexpr (!T::kTwo) issue(std::integral_constant<int, 2 * j + 1>{}, std::integral_constant<int, 2 * MF>{});
        });
        if constexpr (T::kTwo) {
#pragma unroll
            for (int f = 0; f < NF; ++f)
#pragma unroll
                for (int j = 0; j < MF; ++j) pin(acc[f][j]);
            __builtin_amdgcn_s_setprio(0);
            if (wm == 0) landed(nc, k + 1);
            lds_barrier();
        }
        wbuf = wbuf == NS - 1 ? 0 : wbuf + 1;
        if (k & 1) abuf = abuf == NA - 1 ? 0 : abuf + 1;
    };
    if constexpr (T::kTwo) {
        landed(Next{}, 0);
        lds_barrier();
        if (wm != 0) lds_barrier();                      // half a step behind
    }
    int k = 0;
    const int first = min(4, K128);
    for (; k < first; ++k) step(Next{}, Next{}, k);
    for (; k + 8 <= K128; k += 4) {                      // every DMA of these steps exists: the last reaches step k + 7
        step(std::integral_constant<int, 0>{}, std::integral_constant<int, 1>{}, k);
        step(std::integral_constant<int, 1>{}, std::integral_constant<int, 2>{}, k + 1);
        step(std::integral_constant<int, 2>{}, std::integral_constant<int, 3>{}, k + 2);
        step(std::integral_constant<int, 3>{}, std::integral_constant<int, 0>{}, k + 3);
    }
    for (; k < K128; ++k) step(Next{}, Next{}, k);
    if constexpr (T::kTwo)
        if (wm == 0) lds_barrier();
    // The matrix unit writes its result after the instruction, and a read of it before then is not held up: the
    // compiler counts the wait states, but was seen to count too few where branches around the DMAs come between
    // (element 15 of an accumulator read stale).  Nothing reads an accumulator before this.
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int j = 0; j < MF; ++j) asm volatile("s_nop 15\n\ts_nop 3" : "+v"(acc[f][j]));
}

// The wave's outputs through its part of LDS, 32 activation rows at a time, so that they leave as 16-byte pieces of
// whole row segments (64 bytes to 384; stored straight from the accumulators, 8 bytes of each of 32 rows at a time, they
// took as long as the loop: 34 us of 132).  row(r): the output row of the wave's activation row r, below 0: none.
template <int MF, int NF, bool BF, class Row>
__device__ __forceinline__ void mx_store(uint8_t* smem, const mx_v16f (&acc)[NF][MF], void* D, int n0, int N, int vec, Row row) {
    constexpr int kSize = BF ? 2 : 4, kPer = 16 / kSize, kRow = 32 * NF * kSize, kStride = kRow + 16, kPieces = kRow / 16;
    const int lane = threadIdx.x & 63;
    uint8_t* buf = smem + (threadIdx.x >> 6) * 32 * kStride;
    __syncthreads();                                     // every wave is done with the operands
#pragma unroll
    for (int j = 0; j < MF; ++j) {
#pragma unroll
        for (int f = 0; f < NF; ++f)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                uint8_t* d = buf + (lane & 31) * kStride + (32 * f + 8 * e + 4 * (lane >> 5)) * kSize;
                const mx_v16f& v = acc[f][j];
                if constexpr (BF) *(uint2*)d = make_uint2(mx_bf16x2(v[4 * e], v[4 * e + 1]), mx_bf16x2(v[4 * e + 2], v[4 * e + 3]));
                else *(mx_v4f*)d = mx_v4f{v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]};
            }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");      // the wave's own writes, read by its other lanes
#pragma unroll
        for (int i = 0; i < 32 * kPieces / 64; ++i) {
            const int p = lane + 64 * i, r = p / kPieces, c = p - r * kPieces, n = n0 + c * kPer;
            const uint4 v = *(const uint4*)(buf + r * kStride + c * 16);
            const int64_t m = row(32 * j + r);
            if (m < 0 || n >= N) continue;
            uint8_t* d = (uint8_t*)D + ((size_t)m * N + n) * kSize;
            if (vec) {
                *(uint4*)d = v;
            } else {
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int q = 0; q < kPer; ++q)
                    if (n + q < N) {
                        if constexpr (BF) ((uint16_t*)d)[q] = (uint16_t)(w[q >> 1] >> (16 * (q & 1)));
                        else ((uint32_t*)d)[q] = w[q];
                    }
            }
        }
        asm volatile("" ::: "memory");                   // reads before the next rows' writes (LDS is in order)
    }
}

template <int MF, int NF, int WM, int WN, int NS, int NA, bool BF>
__global__ void __launch_bounds__(64 * WM * WN, 2) k_gemm_mxfp4(const uint8_t* __restrict__ W, qmm_xmx x, void* __restrict__ D, int M, int N, int K128,
                                                                int mtiles, int panel, int vec) {
    using T = MxTile<MF, NF, WM, WN, NS, NA>;
    extern __shared__ __align__(16) uint8_t smem[];
    // workgroup i runs on XCD i % 8: each XCD takes a contiguous range of tiles, rows fastest, so that the
    // tiles it runs together share weight strips in its L2
    const uint32_t total = gridDim.x, xcd = blockIdx.x & 7, q = total >> 3, rem = total & 7;
    const uint32_t t = xcd * q + min(xcd, rem) + (blockIdx.x >> 3);
    const uint32_t ntiles = total / (uint32_t)mtiles, pan = t / (panel * ntiles), left = t - pan * panel * ntiles;
    const uint32_t pm = min((uint32_t)panel, (uint32_t)mtiles - pan * panel);
    const int m0 = (int)(pan * panel + left % pm) * T::kRows, n0 = (int)(left / pm) * T::kCols;
    mx_v16f acc[NF][MF];
    mx_tile<MF, NF, WM, WN, NS, NA>(smem, W, x, n0 / 16, (N + 15) / 16, K128, [&](int r) { return min(m0 + r, M - 1); }, acc);
    const int wave = threadIdx.x >> 6, mw = m0 + 32 * MF * (wave / WN);
    mx_store<MF, NF, BF>(smem, acc, D, n0 + 32 * NF * (wave % WN), N, vec, [&](int r) { return mw + r < M ? (int64_t)(mw + r) : -1; });
}

// Grouped: workgroup (tile of one expert's rows, block of 128 outputs); a tile's rows 64 at a time, with as
// many 32-row fragments as they need.
constexpr int kMoeNS = 4, kMoeNA = 3, kMoeCols = 128, kMoeRows = 64;

template <int MF, bool BF>
__device__ __forceinline__ void moe_rows(uint8_t* smem, const uint8_t* We, qmm_xmx x, const int* rowtab, int k0, int n, int n0, void* D, int N, int K128,
                                         int vec) {
    mx_v16f acc[1][MF];
    mx_tile<MF, 1, 1, 4, kMoeNS, kMoeNA>(smem, We, x, n0 / 16, (N + 15) / 16, K128, [&](int r) {
        const int k = k0 + min(r, n - 1);
        return rowtab ? rowtab[k] : k;
    }, acc);
    mx_store<MF, 1, BF>(smem, acc, D, n0 + 32 * (int)(threadIdx.x >> 6), N, vec, [&](int r) { return r < n ? (int64_t)(k0 + r) : -1; });
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
        __syncthreads();                                 // the ring is filled again
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

constexpr int64_t kPanelBytes = 5 << 19;

template <int MF, int NF, int WM, int WN, int NS, int NA>
int launch_gemm(const void* W, qmm_xmx x, void* D, int dtype, int M, int N, int K128, hipStream_t s) {
    using T = MxTile<MF, NF, WM, WN, NS, NA>;
    static_assert(T::kLds <= 160 * 1024, "LDS of a CU");
    const int64_t mt = ((int64_t)M + T::kRows - 1) / T::kRows, nt = ((int64_t)N + T::kCols - 1) / T::kCols;
    if (mt * nt > 0x7fffffff) return QMM_ERR_SHAPE;
    const dim3 grid((unsigned)(mt * nt)), block(64 * T::kWaves);
    const int64_t fit = std::max<int64_t>(1, kPanelBytes / ((int64_t)T::kRows * K128 * 64)), np = (mt + fit - 1) / fit;
    const int panel = (int)((mt + np - 1) / np);
    if (dtype == QMM_BF16)
        hipLaunchKernelGGL((k_gemm_mxfp4<MF, NF, WM, WN, NS, NA, true>), grid, block, T::kLds, s, (const uint8_t*)W, x, D, M, N, K128, (int)mt, panel,
                           vec16_out(D, dtype, N));
    else
        hipLaunchKernelGGL((k_gemm_mxfp4<MF, NF, WM, WN, NS, NA, false>), grid, block, T::kLds, s, (const uint8_t*)W, x, D, M, N, K128, (int)mt, panel,
                           vec16_out(D, dtype, N));
    QMM_LAUNCH_CHECK();
    return QMM_OK;
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
    const auto tiles = [&](int bm, int bn) { return (((int64_t)M + bm - 1) / bm) * (((int64_t)N + bn - 1) / bn); };
    if (tiles(192, 384) >= 200) return launch_gemm<3, 3, 2, 4, 3, 2>(W, x, D, dtype, M, N, K128, s);
    if (tiles(128, 128) >= 256) return launch_gemm<2, 2, 2, 2, 3, 2>(W, x, D, dtype, M, N, K128, s);
    return launch_gemm<2, 1, 1, 4, 4, 2>(W, x, D, dtype, M, N, K128, s);
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
    constexpr size_t lds = MxTile<2, 1, 1, 4, kMoeNS, kMoeNA>::kLds;
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
