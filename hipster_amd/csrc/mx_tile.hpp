// mx_tile.hpp -- the two cores of the MXFP4 GEMMs (mx_gemm.hip) and the way their outputs leave.
//
// Both run on v_mfma_scale_f32_32x32x64_f8f6f4 and add an output's products in the same order (one chain over K), so
// a result does not depend on which core or tile ran.  On an idle chip an instruction takes 14.5 ns; with every CU
// busy 23 (the card lowers its clock for power), 6.2 PFLOP/s in all: the ceiling of a large product.
//
//   mx_tile_reg   32 MF x 128 NF outputs, four waves.  What bounds a step (128 values) of few tiles is how far
//                 ahead its bytes are asked for: memory answers after one to two microseconds, a step multiplies for a
//                 fraction of one.  Weights go straight from memory to the operand registers, D - 1 steps ahead (a
//                 strip belongs to one wave; through LDS it would take two thirds of its bandwidth).  Activations,
//                 which the waves share, come two steps at a time (a pair: 128 bytes of a row, whole cache lines),
//                 D steps ahead in registers, then through LDS: three buffers, so that one barrier a pair
//                 suffices.  LDS reads run two 32-row fragments ahead of their products, across steps.
//                 65 rows x 5120 x 5120: 10.8 us (29 for the other core's best tile); 300 x 17408 x 5120: 26 with weights
//                 from memory, 23.5 from the last-level cache.  Taken apart when it took 28.5: 23.9 with weights that hit the L1,
//                 20.7 without LDS reads too, 19.7 without LDS writes, 17.7 with products, launch and outputs alone: 204 tiles
//                 of 128 x 256 on 256 CUs, 384 rows multiplied for 300, one wave a SIMD.
//   mx_tile_dma   64 MF x 128 NF outputs, eight waves, for many rows.  Both operands by DMA (global_load_lds):
//                 activations by pairs into two buffers, weights step by step into a ring of NS, scales by groups of
//                 four steps.  The waves run as two halves (the rows' halves, one wave of each on every SIMD) half a step
//                 apart: while one half reads its operands from LDS and starts its DMAs, the other multiplies, and a
//                 barrier ends each phase.  2048 x 17408 x 5120, a new weight each call: 101 to 105 us (3.5 PFLOP/s) against
//                 129 for the best tile of mx_tile_reg; without its DMAs it takes 71, without products and LDS reads 72.
//
// LDS holds an activation row's 16-byte chunk c at chunk c ^ a_swz(row): reads of 16 rows' chunk are free of bank
// conflicts for any row alignment of 32.
#pragma once
#include "mx.hpp"

#include <type_traits>

namespace qmm {

__device__ __forceinline__ int a_swz(int row) { return ((row >> 1) & 7) ^ ((row & 1) << 2); }

template <int I, int N, class F>
__device__ __forceinline__ void static_for(F f) {
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        static_for<I + 1, N>(f);
    }
}

// The accumulator exists here (no instruction): the compiler would otherwise gather the products, which touch no
// memory, at the end of the loop, and hold every step's operands until then.  AGPR: where it lives in the second half
// of the 512 registers that a wave has when it is alone on its SIMD.
template <bool AGPR>
__device__ __forceinline__ void pin(mx_v16f& v) {
    if constexpr (AGPR) asm volatile("" : "+a"(v));
    else asm volatile("" : "+v"(v));
}

// The matrix unit writes its result after the instruction, and a read of it before then is not held up: the
// compiler counts the wait states, but was seen to count too few where branches around inline assembly came
// between (element 15 of an accumulator read stale).  Nothing reads an accumulator before this.
template <bool AGPR, int NF, int MF>
__device__ __forceinline__ void settle(mx_v16f (&acc)[NF][MF]) {
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int j = 0; j < MF; ++j) {
            if constexpr (AGPR) asm volatile("s_nop 15\n\ts_nop 3" : "+a"(acc[f][j]));
            else asm volatile("s_nop 15\n\ts_nop 3" : "+v"(acc[f][j]));
        }
}

// ---- weights in registers ----
template <int MF, int NF>
struct MxReg {
    static constexpr int kThreads = 256;
    static constexpr int kRows = 32 * MF, kCols = 128 * NF;
    static constexpr int kCodes = kRows * 128, kStage = kCodes + kRows * 8;
    static constexpr int kStoreLds = 4 * 32 * (128 * NF + 16);
    static constexpr int kLds = 3 * kStage > kStoreLds ? 3 * kStage : kStoreLds;
};

struct AsItIs { __device__ int operator()(int r) const { return r; } };

// fit(rows(r)): the activation row of tile row r (rows may load from a table: all of them first, then what fit does with them,
// or each load would be waited for by itself).  acc[f][j]: weight rows 32 f.., activation rows 32 j.. of this wave
template <int MF, int NF, int D, bool AGPR, class Rows, class Fit = AsItIs>
__device__ __forceinline__ void mx_tile_reg(uint8_t* smem, const uint8_t* W, qmm_xmx x, int strip0, int nstrips, int K128, Rows rows, mx_v16f (&acc)[NF][MF],
                                            Fit fit = Fit{}) {
    using T = MxReg<MF, NF>;
    static_assert(D == 4 || D == 8, "the ring of weights turns with the groups of four steps");
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
    const int last = K128 - 1, G = mx_groups(K128);

    // weights: from the wave's first strip, this lane's row and block `half` of each 32 rows
    const uint32_t sb = mx_strip_bytes(K128), slot = (uint32_t)(half * 16 + (lane & 15));
    const int s0 = min(strip0 + 2 * wave * NF, nstrips - 1);
    const uint8_t* wbase = W + (size_t)s0 * sb;
    uint32_t woff[NF], soff[NF];
#pragma unroll
    for (int f = 0; f < NF; ++f) {
        const uint32_t s = (uint32_t)(min(s0 + 2 * f + ((lane >> 4) & 1), nstrips - 1) - s0) * sb;
        woff[f] = s + slot * 16u;
        soff[f] = s + (uint32_t)K128 * 1024u + slot * 4u;
    }
    uint4 w[D][NF][2];
    uint32_t ws[NF][2], wsn[NF][2];
    auto load_w = [&](uint4 (&d)[NF][2], int k, int i) {                   // piece i of 2 NF
        d[i >> 1][i & 1] = ld16(wbase + (uint32_t)min(k, last) * 1024u + woff[i >> 1] + (i & 1) * 512u);
    };
    auto load_ws = [&](uint32_t (&d)[NF][2], int g) {
        const uint8_t* p = wbase + (uint32_t)min(g, G - 1) * 256u;
#pragma unroll
        for (int f = 0; f < NF; ++f) { d[f][0] = *(const uint32_t*)(p + soff[f]); d[f][1] = *(const uint32_t*)(p + soff[f] + 128u); }
    };

    // activations: chunk tid % 8 of the rows tid / 8 + 32 i, and the scales of row tid / 2 in step tid % 2 of a pair,
    // and of row 128 + tid / 2 where the tile has more than 128
    const int cj = tid & 7;
    const uint8_t* qp[MF];
    int qr[MF];
#pragma unroll
    for (int i = 0; i < MF; ++i) qr[i] = rows((tid >> 3) + 32 * i);
    constexpr int NE = (2 * T::kRows + 255) / 256;
    int es[NE], er[NE];
    const uint8_t* ep[NE];
#pragma unroll
    for (int i = 0; i < NE; ++i) {
        es[i] = min(tid + 256 * i, 2 * T::kRows - 1);    // beyond: the last one again
        er[i] = rows(es[i] >> 1);
    }
#pragma unroll
    for (int i = 0; i < MF; ++i) qp[i] = x.q + (size_t)fit(qr[i]) * K128 * 64 + (cj & 3) * 16;
#pragma unroll
    for (int i = 0; i < NE; ++i) ep[i] = x.e + (size_t)fit(er[i]) * K128 * 4;
    constexpr int NP = D / 2;                            // pairs in flight
    uint4 pa[NP][MF];
    uint32_t pe[NP][NE];
    auto load_a = [&](uint4 (&d)[MF], int p, int i) { d[i] = ld16(qp[i] + (uint32_t)min(2 * p + (cj >> 2), last) * 64u); };
    auto load_as = [&](uint32_t (&e)[NE], int p) {
#pragma unroll
        for (int i = 0; i < NE; ++i) e[i] = *(const uint32_t*)(ep[i] + (uint32_t)min(2 * p + (es[i] & 1), last) * 4u);
    };
    auto put_a = [&](const uint4 (&v)[MF], int buf, int i) {
        const int row = (tid >> 3) + 32 * i;
        *(uint4*)(smem + buf * T::kStage + row * 128 + ((cj ^ a_swz(row)) << 4)) = v[i];
    };
    auto put_as = [&](const uint32_t (&e)[NE], int buf) {
#pragma unroll
        for (int i = 0; i < NE; ++i) *(uint32_t*)(smem + buf * T::kStage + T::kCodes + es[i] * 4) = e[i];
    };
    auto load_pair = [&](uint4 (&d)[MF], uint32_t (&e)[NE], int p) {
#pragma unroll
        for (int i = 0; i < MF; ++i) load_a(d, p, i);
        load_as(e, p);
    };
    // this lane's part of fragment j in step parity s of a buffer: two blocks' codes, the four scale bytes
    struct Frag { uint4 c0, c1; uint32_t s; };
    const int fr = lane & 31, sw = a_swz(fr);            // rows 32 apart: the same rotation
    const uint32_t at0 = (uint32_t)(fr * 128 + ((half ^ sw) << 4)), at1 = (uint32_t)(fr * 128 + (((half + 2) ^ sw) << 4));
    auto read_a = [&](int buf, int s, int j) {
        const uint8_t* d = smem + buf * T::kStage;
        Frag r;
        r.c0 = *(const uint4*)(d + (at0 ^ (64u * s)) + 4096 * j);
        r.c1 = *(const uint4*)(d + (at1 ^ (64u * s)) + 4096 * j);
        r.s = *(const uint32_t*)(d + T::kCodes + fr * 8 + 256 * j + 4 * s);
        return r;
    };

#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int j = 0; j < MF; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[f][j][e] = 0.f;

    load_ws(ws, 0);
#pragma unroll
    for (int k = 0; k < D; ++k) {                        // in the order of their use: loads return in the order of issue
        if (k % 2 == 0) load_pair(pa[k / 2], pe[k / 2], k / 2);
        if (k == D - 1) break;
#pragma unroll
        for (int i = 0; i < 2 * NF; ++i) load_w(w[k], k, i);
    }
#pragma unroll
    for (int i = 0; i < MF; ++i) put_a(pa[0], 0, i);
    put_as(pe[0], 0);
    load_pair(pa[0], pe[0], NP);
    lds_barrier();

    int buf = 0;                                         // of the current pair
    auto after = [](int b) { return b == 2 ? 0 : b + 1; };
    constexpr int kAhead = MF > 1 ? 2 : 1;               // fragments read ahead (fragments of one step follow the last step's)
    Frag fa[MF + kAhead];
    static_for<0, kAhead>([&](auto jc) { fa[jc.value] = read_a(0, jc.value / MF, jc.value % MF); });
    // Step k of ring slot U (k % D).  A wave issues some four instructions in the time of a product, so the rest of the
    // step lies between the products: after the first of a fragment the reads of a later one, after its last the
    // activations' part.  The weights' loads come after the step's first product, except in a wave that is
    // alone on its SIMD, which spreads them over the fragments (128 x 256: 44 us against 47 at 2048 x 5120 x 5120; two
    // waves a SIMD take 35.6 that way at 100 x 5120 x 17408, 32.4 so).
    constexpr int kMeet = MF > 2 ? MF - 3 : -1;          // the fragment of an odd step after which the waves meet
    auto step = [&](auto uc, int k) {
        constexpr int U = decltype(uc)::value, S = U & 3, P = ((U >> 1) + 1) % NP;
        static_for<0, MF>([&](auto jc) {
            constexpr int j = decltype(jc)::value, n = j + kAhead;
            const uint32_t sa = fa[j].s >> (8 * half);   // the lane's two in bytes 0 and 2
            static_for<0, 2 * NF>([&](auto ic) {
                constexpr int i = decltype(ic)::value, f = i % NF, h = i / NF;
                acc[f][j] = mx_mfma32<S, 2 * h>(w[U][f][h], h ? fa[j].c1 : fa[j].c0, acc[f][j], ws[f][h], sa);
                pin<AGPR>(acc[f][j]);
                __builtin_amdgcn_sched_barrier(0);
                // the fragment kAhead on: of this step, or of the next one (in the next buffer after the second of a pair)
                if constexpr (i == 0) {
                    if constexpr (n < MF) fa[n] = read_a(buf, U & 1, n);
                    else if constexpr ((U & 1) == 1) fa[n] = read_a(after(buf), 0, n - MF);
                    else if constexpr (n - MF < MF) fa[n] = read_a(buf, 1, n - MF);
                }
                if constexpr (AGPR ? i == NF : i == 0 && j == 0) {
                    constexpr int lo = AGPR ? 2 * NF * j / MF : 0, hi = AGPR ? 2 * NF * (j + 1) / MF : 2 * NF;
#pragma unroll
                    for (int l = lo; l < hi; ++l) load_w(w[(U + D - 1) % D], k + D - 1, l);
                    if constexpr (S == 1 && j == 0) load_ws(wsn, (k >> 2) + 1);
                }
                if constexpr (i == 2 * NF - 1 && (U & 1) == 0) {
                    put_a(pa[P], after(buf), j);         // pair k / 2 + 1
                    load_a(pa[P], (k >> 1) + 1 + NP, j);
                    if constexpr (j == MF - 1) {
                        put_as(pe[P], after(buf));
                        load_as(pe[P], (k >> 1) + 1 + NP);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            });
            if constexpr ((U & 1) == 1 && j == kMeet) lds_barrier();             // opens the next pair
        });
        static_for<0, kAhead>([&](auto jc) { fa[jc.value] = fa[MF + jc.value]; });
        if constexpr ((U & 1) == 1) buf = after(buf);
        else if constexpr (kMeet < 0) lds_barrier();
        if constexpr (S == 3) {
#pragma unroll
            for (int f = 0; f < NF; ++f) { ws[f][0] = wsn[f][0]; ws[f][1] = wsn[f][1]; }
        }
    };
    int k = 0;
    for (; k + D <= K128; k += D) static_for<0, D>([&](auto uc) { step(uc, k + uc.value); });
    static_for<0, D - 1>([&](auto uc) {
        if (k + uc.value < K128) step(uc, k + uc.value);
    });
    settle<AGPR>(acc);
}

// ---- both operands by DMA ----
template <int MF, int NF, int NS>
struct MxDma {
    static constexpr int NA = 2, kWaves = 8, kThreads = 512, kRows = 64 * MF, kCols = 128 * NF;
    static constexpr int per(int pieces) { return (pieces + kWaves - 1) / kWaves; }
    // DMAs (1 KB each): of a pair's activations, of a step's weights, of a group's scales; and per wave
    static constexpr int kAPieces = kRows / 8, kWPieces = kCols / 16, kRowSc = (kRows + 63) / 64, kScPieces = kRowSc + (kCols + 63) / 64;
    static constexpr int PA = per(kAPieces), PW = per(kWPieces), PS = per(kScPieces);
    static constexpr int kABytes = kAPieces * 1024, kWBytes = kWPieces * 1024, kScBytes = kScPieces * 1024;
    static constexpr int kWAt = NA * kABytes, kScAt = kWAt + NS * kWBytes, kLoopLds = kScAt + 2 * kScBytes;
    static constexpr int kStoreLds = kWaves * 32 * (128 * NF + 16), kLds = kLoopLds > kStoreLds ? kLoopLds : kStoreLds;
    // what a wave issues in step j (mod 4): scales of the next group, a pair, a step of weights, in this order
    static constexpr int issued(int j) { return PW + ((j & 1) == 0 ? PA : 0) + ((j & 3) == 0 ? PS : 0); }
    static constexpr int issued(int from, int to) { return from > to ? 0 : issued(from) + issued(from + 1, to); }
    // DMAs younger than those that step k (mod 4, plus a multiple of 4) reads
    static constexpr int younger(int k) {
        const int w = issued(k - NS + 2, k - 1), a = PW + issued(k - 2 * (NA - 1) + 1, k - 1);
        return (k & 1) == 0 && a < w ? a : w;
    }
    static_assert(NS >= 3 && NS <= 4, "the waits below hold for these");
};

// s_waitcnt vmcnt(n)
template <int N>
__device__ __forceinline__ void vm_wait() {
    static_assert(N >= 0 && N < 64, "vmcnt has six bits");
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}

// the value exists here, in registers (no instruction)
__device__ __forceinline__ void pin(uint32_t& v) { asm volatile("" : "+v"(v)); }
__device__ __forceinline__ void pin(uint4& a, uint4& b) {
    asm volatile("" : "+v"(a.x), "+v"(a.y), "+v"(a.z), "+v"(a.w), "+v"(b.x), "+v"(b.y), "+v"(b.z), "+v"(b.w));
}
// rows(r): the activation row of tile row r.  acc[f][j]: weight rows 32 f.., activation rows 32 j.. of this wave
template <int MF, int NF, int NS, class Rows>
__device__ __forceinline__ void mx_tile_dma(uint8_t* smem, const uint8_t* W, qmm_xmx x, int strip0, int nstrips, int K128, Rows rows, mx_v16f (&acc)[NF][MF]) {
    using T = MxDma<MF, NF, NS>;
    constexpr int NA = T::NA;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wn = wave & 3, wm = wave >> 2, half = lane >> 5;
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
        for (int i = tid; i < T::kRows * K128; i += T::kThreads) {
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
        const int an = abuf == 0 ? NA - 1 : abuf - 1, wn_ = wbuf == 0 ? NS - 1 : wbuf - 1;
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
#pragma unroll
        for (int j = 0; j < MF; ++j) read_a(j);
        // the step's DMAs: the next group's scales, a pair, a step of weights
        if constexpr (S <= 0)
            if (kSteady || ((k & 3) == 0 && k + 4 < K128))
#pragma unroll
                for (int i = 0; i < T::PS; ++i) issue_s(i, g + 1);
        if constexpr (!kSteady || (S & 1) == 0)
            if (kSteady || ((k & 1) == 0 && k + 2 * (NA - 1) < K128))
#pragma unroll
                for (int i = 0; i < T::PA; ++i) issue_a(i, (k >> 1) + NA - 1, an);
        if (kSteady || k + NS - 1 < K128)
#pragma unroll
            for (int i = 0; i < T::PW; ++i) issue_w(i, wn_);
        // the compiler would move the reads and the products to where they suit it: they stay in their phases
#pragma unroll
        for (int f = 0; f < NF; ++f) pin(w[f][0], w[f][1]);
#pragma unroll
        for (int j = 0; j < MF; ++j) { pin(a[j][0], a[j][1]); pin(sa[j]); }
        if (wm != 0) landed(nc, k + 1);
        lds_barrier();
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int j = 0; j < MF; ++j) {
#pragma unroll
            for (int f = 0; f < NF; ++f) acc[f][j] = mx_mfma32<kSteady ? S : 0, 0>(w[f][0], a[j][0], acc[f][j], ws[f][0], sa[j]);
#pragma unroll
            for (int f = 0; f < NF; ++f) acc[f][j] = mx_mfma32<kSteady ? S : 0, 2>(w[f][1], a[j][1], acc[f][j], ws[f][1], sa[j]);
        }
#pragma unroll
        for (int f = 0; f < NF; ++f)
#pragma unroll
            for (int j = 0; j < MF; ++j) pin<false>(acc[f][j]);
        __builtin_amdgcn_s_setprio(0);
        if (wm == 0) landed(nc, k + 1);
        lds_barrier();
        wbuf = wbuf == NS - 1 ? 0 : wbuf + 1;
        if (k & 1) abuf = abuf == NA - 1 ? 0 : abuf + 1;
    };
    landed(Next{}, 0);
    lds_barrier();
    if (wm != 0) lds_barrier();                          // half a step behind
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
    if (wm == 0) lds_barrier();
    settle<false>(acc);
}

// ---- outputs ----
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

}  // namespace qmm
