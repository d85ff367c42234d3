// attn_prompt.hip -- causal attention of packed prompts, bf16, grouped heads.
//
//   k_attn_prompt   32 query rows a wave, keys and values in tiles of 64 through LDS
//
// Per row: t_j = scale log2(e) q . k_j, o = sum_j 2^(t_j - m) v_j / (sum_j 2^(t_j - m) + 2^(sink log2(e) - m)), in one pass over the keys
// with the running maximum m.  Scores, weights, sums and outputs are f32; a weight is rounded to bf16 (2^-8 of it at most, as the output
// is) as a factor of the second product, the sum of weights takes them unrounded.  Against 64 bits an output is off by 0.0019 to 0.0023 of its
// size, where weights in f32 give 0.0016 to 0.0017 (its own rounding to bf16 among both); weights of more bits would take two or
// three products for one.
//
// The floor is the matrix units': 4 dim operations a visible pair.  Products run on the 32 x 32 x 16 bf16 instruction with keys as
// rows: S^T = K Q^T, O^T = V^T P^T.  A lane of S^T holds 16 of 32 keys of one query row: the row's maximum and sum are its own registers and
// one exchange with lane l ^ 32, and what the second product takes of P^T from a lane is just what it has, so P never leaves its
// registers.  V^T is read from LDS by the transposing read, four keys of 16 dims at a time.
//
// Tiles come by DMA into one of two buffers while the other is worked on: two barriers a tile.  Lines of a tile's rows are permuted
// (key_turn, val_turn), so that what one instruction reads lies in different banks (counted: no conflicts).
//
// 8192 rows, 32 heads on 8 of 128 dims: 519 to 547 us (1005 to 1060 TFLOP/s; a library product of bf16 that is bound by the card's power
// reaches 1250).  Counted: a CU is busy for 906 000 cycles whatever the time (launches of 547 to 616 us: the clock falls from 1.8 to 1.55 GHz
// under load), 3480 for a tile of both its workgroups.  Of a SIMD's the matrix unit takes 2048 (59 %) and vector instructions 2120
// (61 %): neither is full, as two waves a SIMD with two barriers a tile leave both waiting.  64 dims, 64 heads 631 us: vector instructions 88 %,
// matrix unit 49 %, so bound by the softmax, as much a pair for half the products.  256 dims, 16 heads 622 to 637 us: 41 and 39 %, one
// wave a SIMD does one mostly after the other.  2048 rows of 128 dims 50 to 55 us: the last rows' chain of 32 tiles.
#include "attn.hpp"

#include <algorithm>
#include <type_traits>

namespace qmm {
namespace {

constexpr int kWaves = 4, kRows = 32 * kWaves;           // q rows of a workgroup
constexpr int kParts = 8;                                // at most
constexpr int kTile = 64;                                // keys of a tile
constexpr float kSlack = 8.f;                            // a maximum may fall behind by a factor of 2^8: weights are then below 2^8, as exact
constexpr int kMaxLd = 1 << 24;                          // a tile's byte offsets stay in 32 bits

struct PromptArgs {
    const uint16_t *q, *k, *v;
    uint16_t* out;
    const int *cuq, *cuk;
    const float* sinks;
    size_t ldq, ldo;
    uint32_t ldk, ldv;
    float scale;                                         // its magnitude times log2(e), not 0
    uint32_t flip;                                       // signs of two values of q: its sign
    int n, window, rows, krows, heads, share, tiles;     // tiles: of q rows, at most
    int parts;                                           // that a tile's keys are cut into
    float* part;                                         // [tiles][heads][parts][D / 4][128 rows][4], with more than one
    float2* ml;                                          // [tiles][heads][parts][128 rows]: m, l
};

__device__ __forceinline__ float swap_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float swap_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// The t-th tile of 128 q rows (all lanes alike): its sequence's rows q0 .. q0 + m - 1 and keys k0 .. k0 + n - 1, its first row r0 of
// them.  false: there are fewer tiles.  The wave adds up 64 sequences' tiles at a time.
struct Tiled { int q0, m, k0, n, r0; };
__device__ __forceinline__ bool find_tile(const PromptArgs& a, int t, Tiled& w) {
    const int lane = threadIdx.x & 63;
    const int* const cuk = a.cuk ? a.cuk : a.cuq;
    int before = 0;
    for (int base = 0; base < a.n; base += 64) {
        const int at = base + lane;
        int q0 = 0, m = 0, k0 = 0, n = 0;
        if (at < a.n) {
            q0 = within(a.cuq[at], a.rows);
            m = max(within(a.cuq[at + 1], a.rows) - q0, 0);
            k0 = within(cuk[at], a.krows);
            n = max(within(cuk[at + 1], a.krows) - k0, 0);
        }
        const int tiles = (m + kRows - 1) / kRows, upto = (int)wave_upto((uint32_t)tiles);
        const unsigned long long behind = __ballot(before + upto > t);
        if (behind) {
            const int l = __builtin_ctzll(behind);
            w = {__builtin_amdgcn_readlane(q0, l), __builtin_amdgcn_readlane(m, l), __builtin_amdgcn_readlane(k0, l), __builtin_amdgcn_readlane(n, l),
                 __builtin_amdgcn_readfirstlane((t - before - __builtin_amdgcn_readlane(upto - tiles, l)) * kRows)};
            return w.r0 >= 0 && w.r0 < w.m;              // false only where so many spans overlap that their tiles' count wrapped
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

// the piece that row r's piece p lies at is p ^ turn: 16 rows' pieces of keys in different 16 bytes of 256, and 4 rows' 4 pieces of values
template <int D>
__device__ __forceinline__ int key_turn(int r) { return D == 64 ? (r >> 1) & 7 : r & 15; }
template <int D>
__device__ __forceinline__ int val_turn(int r) { return D == 64 ? 4 * ((r >> 1) & 1) : 4 * (r & 3); }

// dma16s without a claim on memory: the compiler may move its own LDS reads past it (they are of other buffers; barriers order the rest)
__device__ __forceinline__ void dma16q(const void* base, uint32_t voff, uint32_t lds) {
    asm volatile(QMM_VMEM_ASM_GUARD "global_load_lds_dwordx4 %0, %1" : : "v"(voff), "s"(base), "{m0}"(lds));
}
// s_waitcnt vmcnt(n): at most n of the wave's DMAs are under way
template <int N>
__device__ __forceinline__ void wait_dma() { asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory"); }

template <int D>
__global__ void __launch_bounds__(64 * kWaves, D == 256 ? 1 : 2) k_attn_prompt(PromptArgs a) {
    constexpr int S = D / 16, DT = D / 32, kRow = 2 * D, kBytes = kTile * kRow;
    extern __shared__ __align__(16) uint8_t smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, kg = lane >> 5;

    // the last tiles first: they see the most keys
    const uint32_t id = blockIdx.x, turn = id / (uint32_t)a.heads;
    // Successive workgroups run on successive dies of eight, each with a cache of its own: a die gets successive heads, which share keys
    // and values (16 prompts of 1024 and fewer, 32 heads on 8 of 128: 121 us, heads in turn 124; 2048 rows 53.5 and 54.5; 256 dims 1 % slower).
    const int i8 = (int)(id - turn * a.heads), h = a.heads % 8 ? i8 : (i8 % 8) * (a.heads / 8) + i8 / 8, hk = h / a.share;
    const int part = (int)(turn % (uint32_t)a.parts), t = a.tiles - 1 - (int)(turn / (uint32_t)a.parts);
    Tiled w;
    if (!find_tile(a, t, w)) return;
    const int q0 = w.q0, m = w.m, k0 = w.k0, n = w.n, r0 = w.r0;
    const int shift = n - m;                             // position of row 0

    // this lane's row
    const int i = r0 + 32 * wave + col;
    const bool live = i < m;
    const int pos = min(i, m - 1) + shift;
    const int lo = a.window > 0 && pos >= a.window ? pos - a.window + 1 : 0, hi = pos;
    // the wave's and the workgroup's keys
    const int wave_first = min(r0 + 32 * wave, m - 1) + shift, wave_last = min(r0 + 32 * wave + 31, m - 1) + shift;
    const int last = min(r0 + kRows - 1, m - 1) + shift, first = a.window > 0 && r0 + shift >= a.window ? r0 + shift - a.window + 1 : 0;
    const int wave_lo = a.window > 0 && wave_first >= a.window ? wave_first - a.window + 1 : 0;
    const int full_lo = a.window > 0 && wave_last >= a.window ? wave_last - a.window + 1 : 0;       // from here on all rows see

    at_bf8 qf[S];
    {
        const uint16_t* p = a.q + (size_t)(q0 + min(i, m - 1)) * a.ldq + (size_t)h * D + 8 * kg;
#pragma unroll
        for (int s = 0; s < S; ++s) {
            uint4 w = *(const uint4*)(p + 16 * s);
            w.x ^= a.flip; w.y ^= a.flip; w.z ^= a.flip; w.w ^= a.flip;
            qf[s] = __builtin_bit_cast(at_bf8, w);
        }
    }
    // DMA of a tile: 1 KiB an instruction, kTile * kRow / 1024 of each matrix over the waves
    constexpr int kLines = kBytes / 1024 / kWaves, kPieces = kRow / 16, kPerLine = 1024 / kRow;      // rows an instruction
    static_assert(kLines >= 1, "");
    const uint8_t* const kbase = (const uint8_t*)(a.k + (size_t)k0 * a.ldk + (size_t)hk * D);
    const uint8_t* const vbase = (const uint8_t*)(a.v + (size_t)k0 * a.ldv + (size_t)hk * D);
    const uint32_t lds0 = lds_addr(smem);
    // Line j of the wave's of keys (VAL: of values) key0 .. + 63 into buffer `stage`, those past the last as the last.  Its rows are the
    // wave's first ones and j * kPerLine further; where a piece lies goes by the row.
    const int fr = wave * kLines * kPerLine + lane / kPieces, fp = lane % kPieces;
    const uint32_t frk = (uint32_t)fr * a.ldk * 2, frv = (uint32_t)fr * a.ldv * 2;
    auto fetch = [&](auto val, int j, int key0, int stage) {
        constexpr bool VAL = decltype(val)::value;
        const uint32_t ld2 = (VAL ? a.ldv : a.ldk) * 2, last_row = (uint32_t)min(n - 1 - key0, kTile - 1) * ld2;
        const uint32_t row = min((VAL ? frv : frk) + (uint32_t)(j * kPerLine) * ld2, last_row);
        const int turn = VAL ? val_turn<D>(fr + j * kPerLine) : key_turn<D>(fr + j * kPerLine);
        dma16q((VAL ? vbase : kbase) + (size_t)key0 * ld2, row + (uint32_t)((fp ^ turn) * 16),
               lds0 + ((VAL ? 2 : 0) + stage) * kBytes + (wave * kLines + j) * 1024);
    };
    auto fetch_k = [&](int key0, int stage) {
#pragma unroll
        for (int j = 0; j < kLines; ++j) fetch(std::false_type{}, j, key0, stage);
    };
    auto fetch_v = [&](int key0, int stage) {
#pragma unroll
        for (int j = 0; j < kLines; ++j) fetch(std::true_type{}, j, key0, stage);
    };
    // addresses of operands within a tile
    constexpr int KA = D == 64 ? 4 : 8, VA = D == 64 ? 2 : 4;
    uint32_t ka[KA], va[VA];
#pragma unroll
    for (int s = 0; s < KA; ++s) ka[s] = col * kRow + ((2 * s + kg) ^ key_turn<D>(col)) * 16;
#pragma unroll
    for (int d = 0; d < VA; ++d) {
        const int r = 4 * kg + ((lane & 15) >> 2), piece = 4 * d + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
        va[d] = r * kRow + (piece ^ val_turn<D>(r)) * 16 + (lane & 1) * 8;
    }

    int t0 = first / kTile, t1 = last < 0 ? -1 : last / kTile;
    if (a.parts > 1) {                                   // this workgroup's part of them
        const int each = max((t1 - t0 + a.parts) / a.parts, 1);
        t0 += part * each;
        t1 = min(t1, t0 + each - 1);
    }
    mx_v16f o[DT], sc[2];
    float mx, ls, raw;                                   // raw: the largest of sc, unmasked
    // scores of the tile in key buffer `stage`
    auto scores = [&](int stage, mx_v16f (&to)[2], auto between) {
        const uint8_t* const ks = smem + stage * kBytes;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int e = 0; e < 16; ++e) to[u][e] = 0.f;
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const at_bf8 kf = *(const at_bf8*)(ks + ka[s % KA] + u * 32 * kRow + (s / KA) * 256);
                to[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[s], to[u], 0, 0, 0);
                between(u * S + s);
            }
        }
    };
    // a row's largest score of a tile
    auto row_max = [&](const mx_v16f (&v)[2]) {
        float tops[4] = {neg_inf(), neg_inf(), neg_inf(), neg_inf()};
#pragma unroll
        for (int e = 0; e < 32; ++e) tops[e % 4] = fmaxf(tops[e % 4], v[e / 16][e % 16]);
        return swap_max(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])));
    };
    // One tile: its weights from its scores in sc, the next tile's scores (NEXT) beside them, its values' product.  SAFE: values that are
    // not finite are kept out of the products where some row does not see them, as 0 times one is not 0.
    auto tile = [&](int kt, int stage, auto next, auto safe) {
        constexpr bool NEXT = decltype(next)::value, SAFE = decltype(safe)::value;
        const int key0 = kt * kTile;
        const bool whole = key0 + kTile - 1 <= wave_first && key0 >= full_lo;
        if (!whole) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int key = key0 + 32 * u + 8 * (e / 4) + 4 * kg + e % 4;
                    if (key < lo || key > hi) sc[u][e] = neg_inf();
                }
        }
        const float top = (whole ? raw : row_max(sc)) * a.scale;
        if (__ballot(top > mx + kSlack)) {               // the sums go on at the new maximum
            const float now = fmaxf(mx, top), f = __builtin_amdgcn_exp2f(mx - (now == neg_inf() ? 0.f : now));
            ls *= f;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d] *= f;
            mx = now;
        }
        const float base = mx == neg_inf() ? 0.f : mx;
        mx_v16f sn[2];
        // between the products the DMAs of K(kt + 2), into this tile's keys' buffer, and below of V(kt + 1): the CU takes in 64 bytes a
        // cycle, and what is issued faster holds the wave up
        if constexpr (NEXT)
            scores(stage ^ 1, sn, [&](int i) {
                if (i % (2 * S / kLines) == 0) fetch(std::false_type{}, i / (2 * S / kLines), min(kt + 2, t1) * kTile, stage);
            });
        at_bf8 pf[4];
        float sums[4] = {0.f, 0.f, 0.f, 0.f};
        auto weights = [&](int u) {                      // of 32 of the tile's keys
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[u][e], a.scale, -base));
                sums[e % 4] += p;
                pf[2 * u + e / 8][e % 8] = (__bf16)p;
            }
        };
        // half of the weights beside the next tile's scores, half beside the first half of the values' product
        weights(0);
        if constexpr (NEXT) {
            wait_dma<kLines>();
            lds_barrier();                               // V(kt) is there (K(kt + 2) need not be)
        }
        weights(1);
        const uint8_t* const vs = smem + (2 + stage) * kBytes;
        bool odd = false;
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const uint8_t* from = vs + va[d % VA] + s * 16 * kRow + (d / VA) * 256;
                const at_s4 v0 = tr_read(from), v1 = tr_read(from + 8 * kRow);
                at_bf8 vf = __builtin_bit_cast(at_bf8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
                if constexpr (SAFE) {
                    uint4 w = __builtin_bit_cast(uint4, vf);
                    uint32_t* x = (uint32_t*)&w;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const bool l = !whole && (x[e] & 0x7f80u) == 0x7f80u, g = !whole && (x[e] & 0x7f800000u) == 0x7f800000u;
                        odd |= l | g;
                        x[e] = (l ? 0u : x[e] & 0xffffu) | (g ? 0u : x[e] & 0xffff0000u);
                    }
                    vf = __builtin_bit_cast(at_bf8, w);
                }
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pf[s], o[d], 0, 0, 0);
                const int i = s * DT + d;
                if constexpr (NEXT)
                    if (i % (4 * DT / kLines) == 0) fetch(std::true_type{}, i / (4 * DT / kLines), (kt + 1) * kTile, stage ^ 1);
            }
        ls += (sums[0] + sums[1]) + (sums[2] + sums[3]);
        if constexpr (SAFE) {
            if (__ballot(odd))                           // they reach the rows that see their key, and no other
                for (int key = max(key0, wave_lo); key <= min(key0 + kTile - 1, wave_last); ++key) {
                    const int r = key - key0;
                    const bool sees = key >= lo && key <= hi;
#pragma unroll
                    for (int d = 0; d < DT; ++d)
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const int dim = 32 * d + 8 * (e / 4) + 4 * kg + e % 4;
                            const uint32_t x = *(const uint16_t*)(vs + r * kRow + (((dim >> 3) ^ val_turn<D>(r)) * 16) + (dim & 7) * 2);
                            if ((x & 0x7f80u) == 0x7f80u && sees) o[d][e] += bf2f(x);
                        }
                }
        }
        if constexpr (NEXT) {
#pragma unroll
            for (int u = 0; u < 2; ++u) sc[u] = sn[u];
            raw = row_max(sc);
        }
    };
    // All tiles.  Keys are one tile ahead of values: K(t + 2) and V(t + 1) come while tile t is worked on.
    auto tiles = [&](auto safe) {
        mx = neg_inf();
        ls = 0.f;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
        if (t0 > t1) return;
        fetch_k(t0 * kTile, 0);
        fetch_k(min(t0 + 1, t1) * kTile, 1);             // past the last tile it is asked for again: as many are under way at every wait
        fetch_v(t0 * kTile, 0);
        wait_dma<2 * kLines>();
        lds_barrier();                                   // K(t0) is there
        scores(0, sc, [](int) {});
        raw = row_max(sc);
        for (int kt = t0; kt < t1; ++kt) {
            wait_dma<kLines>();
            lds_barrier();                               // K(kt + 1) is there, and all are done with K(kt) and V(kt - 1)
            tile(kt, (kt - t0) & 1, std::true_type{}, safe);
        }
        wait_dma<0>();
        lds_barrier();
        tile(t1, (t1 - t0) & 1, std::false_type{}, safe);
    };
    tiles(std::false_type{});
    // Where all is finite that is it.  A value that is not, at a key that some row of a tile does not see, made that row's sum NaN:
    // once more, with such values kept out (all waves, as they fetch together).
    float z = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) z = __builtin_fmaf(o[d][e], 0.f, z);
    if (__syncthreads_or(!(z == 0.f))) tiles(std::true_type{});

    ls = swap_sum(ls);
    if (!live) return;
    if (a.parts > 1) {
        const size_t at = ((size_t)t * a.heads + h) * a.parts + part;
        const int r = 32 * wave + col;
        if (kg == 0) a.ml[at * kRows + r] = make_float2(mx, t0 > t1 ? -1.f : ls);            // -1: no keys, and nothing behind it
        if (t0 > t1) return;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                *(mx_v4f*)(a.part + ((at * (D / 4) + 8 * d + 2 * e + kg) * kRows + r) * 4) = mx_v4f{o[d][4 * e], o[d][4 * e + 1], o[d][4 * e + 2], o[d][4 * e + 3]};
        return;
    }
    const float f = finish(1.f, ls, mx, a.sinks, h);
    uint16_t* const to = a.out + (size_t)(q0 + i) * a.ldo + (size_t)h * D + 4 * kg;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            *(uint2*)(to + 32 * d + 8 * e) = make_uint2(mx_bf16x2(o[d][4 * e] * f, o[d][4 * e + 1] * f), mx_bf16x2(o[d][4 * e + 2] * f, o[d][4 * e + 3] * f));
}

// The parts of a tile's rows: 32 rows and 32 dims a workgroup, four dims of a row a thread.
template <int D>
__global__ void __launch_bounds__(256) k_attn_prompt_join(PromptArgs a) {
    constexpr int kCuts = 4 * (D / 32);                  // workgroups of a tile
    const uint32_t th = blockIdx.x / kCuts, cut = blockIdx.x % kCuts;
    const int h = (int)(th % (uint32_t)a.heads), t = (int)(th / (uint32_t)a.heads);
    Tiled w0;
    if (!find_tile(a, t, w0)) return;
    const int q0 = w0.q0, r0 = w0.r0;
    const int r = (int)(cut & 3) * 32 + (threadIdx.x & 31), d = (int)(cut >> 2) * 8 + ((int)threadIdx.x >> 5);
    if (r0 + r >= w0.m) return;
    const size_t at = ((size_t)t * a.heads + h) * a.parts;
    float w[kParts], top = neg_inf(), l = 0.f;
#pragma unroll
    for (int p = 0; p < kParts; ++p)
        if (p < a.parts) top = fmaxf(top, a.ml[(at + p) * kRows + r].x);
#pragma unroll
    for (int p = 0; p < kParts; ++p)
        if (p < a.parts) {
            const float2 v = a.ml[(at + p) * kRows + r];
            w[p] = v.y < 0.f ? -1.f : weight(v.x, top);
            l += v.y < 0.f ? 0.f : w[p] * v.y;
        }
    const float f = finish(1.f, l, top, a.sinks, h);
    uint16_t* const to = a.out + (size_t)(q0 + r0 + r) * a.ldo + (size_t)h * D;
    mx_v4f o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int p = 0; p < kParts; ++p)                     // a part without keys has left nothing; one without weight may have left NaN
        if (p < a.parts && !(w[p] < 0.f)) o += w[p] * *(const mx_v4f*)(a.part + (((at + p) * (D / 4) + d) * kRows + r) * 4);
    *(uint2*)(to + 4 * d) = make_uint2(mx_bf16x2(o[0] * f, o[1] * f), mx_bf16x2(o[2] * f, o[3] * f));
}

// tiles of q rows of a call, at most: a sequence's last may be short
int64_t tiles_of(int rows, int nseq) { return nseq == 1 ? ((int64_t)rows + kRows - 1) / kRows : (int64_t)rows / kRows + nseq; }

// Parts that a tile's keys are cut into: one, or where that leaves half the CUs' room without work as many as fill it, of 16 tiles of
// keys at least (an average row's; each part writes and reads its sums, 64 KB for 128 dims).  512 rows behind 7488 keys, 16 heads of
// 256: one part 309 us, four 91; 1024 rows alone, 32 heads of 128, whose parts would be of 8 tiles: one 27, two 31.
// A window leaves a tile of rows window + 127 keys, however many there are.  Below 8 tiles of window (4 of 256 dims, whose tile takes
// twice the time) they stay one part, above parts are of two tiles at least.  In us with one part and with the parts that the keys' number
// would make, at windows of
//                                                            128          256          512         1024         2048
//   128 rows, 8000 keys, 32 heads of 128, 7 parts        12.6  17.3   15.1  20.0   19.3  20.0   27.5  22.8   44.5  27.2
//   512 rows of them, 4 parts                            13.1  30.9   15.6  30.5   19.6  31.3   28.0  34.9   45.2  40.5
//   64 rows, 16000 keys, 8 heads of 64, 8 parts           7.3  11.6    8.9  12.5   12.0  13.3   18.5  14.6   31.0  16.5
//   512 rows, 8000 keys, 16 heads of 256, 4 parts        21.7  31.8   26.4  31.3   34.5  35.0   51.1  38.0   84.2  46.4
int parts_of(int rows, int krows, int nseq, int heads, int dim, int window) {
    const int64_t work = tiles_of(rows, nseq) * heads, room = (int64_t)device_cu_count() * (dim == 256 ? 1 : 2);
    const int64_t keys = std::max<int64_t>((int64_t)krows - rows / 2, 0) / nseq / kTile;
    int64_t parts = std::min<int64_t>({room / std::max<int64_t>(work, 1), keys / 16, kParts});
    if (window > 0) {
        const int64_t seen = ((int64_t)window + kRows - 1 + kTile - 1) / kTile;          // tiles of keys
        parts = window < (dim == 256 ? 4 : 8) * kTile ? 1 : std::min(parts, seen / 2);
    }
    return (int)std::max<int64_t>(parts, 1);
}

size_t ws_of(int64_t tiles, int heads, int parts, int dim) { return parts == 1 ? 0 : (size_t)tiles * heads * parts * kRows * (dim + 2) * sizeof(float); }

template <int D>
int launch(PromptArgs& a, hipStream_t s) {
    constexpr int kLds = 4 * kTile * 2 * D;
    const uint64_t grid = (uint64_t)a.tiles * a.heads * a.parts;
    if (!grid_fits(grid, 64 * kWaves)) return QMM_ERR_SHAPE;
    hipLaunchKernelGGL((k_attn_prompt<D>), dim3((unsigned)grid), dim3(64 * kWaves), kLds, s, a);
    QMM_LAUNCH_CHECK();
    if (a.parts > 1) {
        hipLaunchKernelGGL((k_attn_prompt_join<D>), dim3((unsigned)(a.tiles * a.heads * 4 * (D / 32))), dim3(256), 0, s, a);
        QMM_LAUNCH_CHECK();
    }
    return QMM_OK;
}

}  // namespace
}  // namespace qmm

using namespace qmm;

extern "C" {

size_t qmm_attn_prompt_ws_bytes(int rows, int krows, int nseq, int heads, int dim) {
    if (rows <= 0 || krows <= 0 || nseq <= 0 || heads <= 0 || (dim != 64 && dim != 128 && dim != 256)) return 0;
    return ws_of(tiles_of(rows, nseq), heads, parts_of(rows, krows, nseq, heads, dim, 0), dim);      // of all windows the most
}

int qmm_attn_prompt_bf16(const uint16_t* q, size_t ldq, const uint16_t* k, size_t ldk, const uint16_t* v, size_t ldv, uint16_t* out, size_t ldo,
                         const int32_t* cuq, const int32_t* cuk, int nseq, const qmm_attn* attn, int rows, int krows, int heads, int kv_heads, int dim,
                         void* ws, size_t ws_bytes, void* stream) {
    if (dim != 64 && dim != 128 && dim != 256) return QMM_ERR_SHAPE;
    if (rows < 0 || krows < 0 || nseq < 0 || heads < 1 || kv_heads < 1 || heads > 65536 || heads % kv_heads) return QMM_ERR_SHAPE;
    if (const int st = attn_check(attn)) return st;
    if (rows == 0 || nseq == 0) return QMM_OK;
    if (!q || !out || !cuq || (krows && (!k || !v))) return QMM_ERR_NULL;
    const size_t nq = (size_t)heads * dim, nk = (size_t)kv_heads * dim;
    if (ldq < nq || ldo < nq || ldk < nk || ldv < nk || ldk > kMaxLd || ldv > kMaxLd) return QMM_ERR_SHAPE;
    if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 16) || ((ldq | ldk | ldv | ldo) & 7)) return QMM_ERR_ARG;
    if (!aligned(cuq, 4) || !aligned(cuk, 4)) return QMM_ERR_ARG;
    const int64_t tiles = tiles_of(rows, nseq);
    if (tiles * heads > 0x1fffffff) return QMM_ERR_SHAPE;
    PromptArgs a;
    a.q = q; a.k = k; a.v = v; a.out = out; a.cuq = cuq; a.cuk = cuk; a.sinks = attn->sinks; a.ldq = ldq; a.ldo = ldo;
    a.ldk = (uint32_t)ldk; a.ldv = (uint32_t)ldv;
    // a scale of 0 (all keys weigh the same) as 2^-126: times a masked score, -inf, it is still -inf
    a.scale = fmaxf((float)(fabs((double)attn->scale) * 1.44269504088896340736), 0x1p-126f);
    a.flip = attn->scale < 0.f ? 0x80008000u : 0u;
    a.n = nseq; a.window = attn->window; a.rows = rows; a.krows = krows; a.heads = heads; a.share = heads / kv_heads; a.tiles = (int)tiles;
    a.parts = ws ? parts_of(rows, krows, nseq, heads, dim, attn->window) : 1;
    if (a.parts > 1) {
        if (ws_bytes < ws_of(tiles, heads, a.parts, dim)) return QMM_ERR_WORKSPACE;
        if (!aligned(ws, 16)) return QMM_ERR_ARG;
        a.part = (float*)ws;
        a.ml = (float2*)(a.part + (size_t)tiles * heads * a.parts * kRows * dim);
    }
    hipStream_t s = (hipStream_t)stream;
    switch (dim) {
        case 64: return launch<64>(a, s);
        case 128: return launch<128>(a, s);
        default: return launch<256>(a, s);
    }
}

}  // extern "C"
