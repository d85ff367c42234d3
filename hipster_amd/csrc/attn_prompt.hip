// attn_prompt.hip -- causal attention of packed prompts, bf16, grouped heads.
//
//   k_attn_prompt   32 query rows a wave, keys and values in tiles of 64 through LDS
//
// Per row: t_j = scale log2(e) q . k_j, o = sum_j 2^(t_j - m) v_j / (sum_j 2^(t_j - m) + 2^(sink log2(e) - m)), in one pass over the keys
// with the running maximum m.  Scores, weights, sums and outputs are f32; a weight is rounded to bf16 (2^-9 of it at most, as the output
// is) as a factor of the second product.
//
// Bound by the matrix units: 4 dim operations a visible pair.  Products run on the 32 x 32 x 16 bf16 instruction with keys as
// rows: S^T = K Q^T, O^T = V^T P^T.  A lane of S^T holds 16 of 32 keys of one query row: the row's maximum and sum are its own registers and
// one exchange with lane l ^ 32, and what the second product takes of P^T from a lane is just what it has, so P never leaves its
// registers.  V^T is read from LDS by the transposing read, four keys of 16 dims at a time.
//
// Tiles come by DMA into one of two buffers while the other is worked on: one barrier a tile.  Lines of a tile's rows are permuted
// (16-byte piece p of row r lies at p ^ (r % 8) for keys, p ^ 2 (r % 4) for values), so that eight rows' pieces, or four rows' pairs of
// pieces, lie in different banks.
#include "attn.hpp"

namespace qmm {
namespace {

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
};

__device__ __forceinline__ float swap_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float swap_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// The sequence and the first row in it of the t-th tile of `size` q rows (all lanes alike); false: there are fewer tiles.  The wave
// adds up 64 sequences' tiles at a time.
__device__ __forceinline__ bool find_tile(const int* __restrict__ cu, int n, int rows, int size, int t, int& b, int& row) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int base = 0; base < n; base += 64) {
        const int at = base + lane;
        int tiles = 0;
        if (at < n) tiles = (max(within(cu[at + 1], rows) - within(cu[at], rows), 0) + size - 1) / size;
        int upto = tiles;
        for (int k = 1; k < 64; k <<= 1) {
            const int v = __shfl_up(upto, k, 64);
            if (lane >= k) upto += v;
        }
        const unsigned long long behind = __ballot(before + upto > t);
        if (behind) {
            const int l = __builtin_ctzll(behind);
            b = base + l;
            row = (t - before - (__shfl(upto, l, 64) - __shfl(tiles, l, 64))) * size;
            b = __builtin_amdgcn_readfirstlane(b);
            row = __builtin_amdgcn_readfirstlane(row);
            return true;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

template <int D, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, D == 256 ? 1 : 2) k_attn_prompt(PromptArgs a) {
    constexpr int S = D / 16, DT = D / 32, kRow = 2 * D, kBytes = kTile * kRow, kStage = 2 * kBytes, kSize = 32 * WAVES;
    extern __shared__ __align__(16) uint8_t smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, kg = lane >> 5;

    // the last tiles first: they see the most keys
    const uint32_t id = blockIdx.x;
    const int h = (int)(id % (uint32_t)a.heads), t = a.tiles - 1 - (int)(id / (uint32_t)a.heads), hk = h / a.share;
    int b, r0;
    if (!find_tile(a.cuq, a.n, a.rows, kSize, t, b, r0)) return;
    const int q0 = within(a.cuq[b], a.rows), m = within(a.cuq[b + 1], a.rows) - q0;
    if (r0 < 0 || r0 >= m) return;                       // only where so many spans overlap that their tiles' count wrapped
    const int* const cuk = a.cuk ? a.cuk : a.cuq;
    const int k0 = within(cuk[b], a.krows), n = max(within(cuk[b + 1], a.krows) - k0, 0);
    const int shift = n - m;                             // position of row 0

    // this lane's row
    const int i = r0 + 32 * wave + col;
    const bool live = i < m;
    const int pos = min(i, m - 1) + shift;
    const int lo = a.window > 0 && pos >= a.window ? pos - a.window + 1 : 0, hi = pos;
    // the wave's and the workgroup's keys
    const int wave_first = min(r0 + 32 * wave, m - 1) + shift, wave_last = min(r0 + 32 * wave + 31, m - 1) + shift;
    const int last = min(r0 + kSize - 1, m - 1) + shift, first = a.window > 0 && r0 + shift >= a.window ? r0 + shift - a.window + 1 : 0;
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
    mx_v16f o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
    float mx = neg_inf(), ls = 0.f;

    // DMA of a tile: 1 KiB an instruction, kTile * kRow / 1024 of each matrix over the waves
    constexpr int kLines = kBytes / 1024 / WAVES, kPieces = kRow / 16, kRowsPer = 1024 / kRow;      // rows an instruction
    static_assert(kLines >= 1, "");
    const uint8_t* const kbase = (const uint8_t*)(a.k + (size_t)k0 * a.ldk + (size_t)hk * D);
    const uint8_t* const vbase = (const uint8_t*)(a.v + (size_t)k0 * a.ldv + (size_t)hk * D);
    const uint32_t lds0 = lds_addr(smem);
    auto fetch = [&](int key0, int stage) {              // keys key0 .. + 63, those past the last as the last
        const uint8_t* kp = kbase + (size_t)key0 * a.ldk * 2;
        const uint8_t* vp = vbase + (size_t)key0 * a.ldv * 2;
#pragma unroll
        for (int j = 0; j < kLines; ++j) {
            const int line = wave * kLines + j, r = line * kRowsPer + lane / kPieces, p = lane % kPieces;
            const uint32_t row = (uint32_t)min(r, n - 1 - key0);
            const uint32_t to = lds0 + stage * kStage + line * 1024;
            dma16s(kp, row * a.ldk * 2 + (uint32_t)((p ^ (r & 7)) * 16), __builtin_amdgcn_readfirstlane(to));
            dma16s(vp, row * a.ldv * 2 + (uint32_t)((p ^ (2 * (r & 3))) * 16), __builtin_amdgcn_readfirstlane(to + kBytes));
        }
    };
    // addresses of operands within a tile
    uint32_t ka[4], va[2];
#pragma unroll
    for (int s = 0; s < 4; ++s) ka[s] = col * kRow + (((2 * s) ^ kg ^ (col & 7)) & 7) * 16;
#pragma unroll
    for (int d = 0; d < 2; ++d) {
        const int r = (lane & 15) >> 2, piece = 4 * d + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
        va[d] = (4 * kg + r) * kRow + (piece ^ (2 * r)) * 16 + (lane & 1) * 8;
    }

    const int t0 = first / kTile, t1 = last < 0 ? -1 : last / kTile;
    if (t0 <= t1) fetch(t0 * kTile, 0);
    for (int kt = t0; kt <= t1; ++kt) {
        const int key0 = kt * kTile, stage = (kt - t0) & 1;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        lds_barrier();                                   // the tile is there, and all are done with the other buffer
        if (kt < t1) fetch(key0 + kTile, stage ^ 1);
        if (key0 > wave_last || key0 + kTile <= wave_lo) continue;           // uniform: nothing of it for this wave
        const uint8_t* const ks = smem + stage * kStage;
        const uint8_t* const vs = ks + kBytes;
        mx_v16f sc[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int e = 0; e < 16; ++e) sc[u][e] = 0.f;
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const at_bf8 kf = *(const at_bf8*)(ks + ka[s & 3] + u * 32 * kRow + (s / 4) * 128);
                sc[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[s], sc[u], 0, 0, 0);
            }
        }
        const bool whole = key0 + kTile - 1 <= wave_first && key0 >= full_lo;
        float top = neg_inf();
        if (!whole) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int key = key0 + 32 * u + 8 * (e / 4) + 4 * kg + e % 4;
                    if (key < lo || key > hi) sc[u][e] = neg_inf();
                }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 16; ++e) top = fmaxf(top, sc[u][e]);
        top = swap_max(top) * a.scale;
        if (__ballot(top > mx + kSlack)) {               // the sums go on at the new maximum
            const float now = fmaxf(mx, top), f = __builtin_amdgcn_exp2f(mx - (now == neg_inf() ? 0.f : now));
            ls *= f;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d] *= f;
            mx = now;
        }
        const float base = mx == neg_inf() ? 0.f : mx;
        at_bf8 pf[4];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[u][e], a.scale, -base));
                ls += p;
                pf[2 * u + e / 8][e % 8] = (__bf16)p;
            }
        bool odd = false;                                // a value that is not finite, where some rows may not see it
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const uint8_t* from = vs + va[d & 1] + s * 16 * kRow + (d / 2) * 128;
                const at_s4 v0 = tr_read(from), v1 = tr_read(from + 8 * kRow);
                at_bf8 vf = __builtin_bit_cast(at_bf8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
                if (!whole) {
                    uint4 w = __builtin_bit_cast(uint4, vf);
                    uint32_t* x = (uint32_t*)&w;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const bool l = (x[e] & 0x7f80u) == 0x7f80u, g = (x[e] & 0x7f800000u) == 0x7f800000u;
                        odd |= l | g;
                        x[e] = (l ? 0u : x[e] & 0xffffu) | (g ? 0u : x[e] & 0xffff0000u);
                    }
                    vf = __builtin_bit_cast(at_bf8, w);
                }
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pf[s], o[d], 0, 0, 0);
            }
        if (!whole && __ballot(odd)) {                   // they reach the rows that see their key, and no other
            for (int key = max(key0, wave_lo); key <= min(key0 + kTile - 1, wave_last); ++key) {
                const int r = key - key0;
                const bool sees = key >= lo && key <= hi;
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int dim = 32 * d + 8 * (e / 4) + 4 * kg + e % 4;
                        const uint32_t x = *(const uint16_t*)(vs + r * kRow + (((dim >> 3) ^ (2 * (r & 3))) * 16) + (dim & 7) * 2);
                        if ((x & 0x7f80u) == 0x7f80u && sees) o[d][e] += bf2f(x);
                    }
            }
        }
    }

    ls = swap_sum(ls);
    if (!live) return;
    float f;
    if (a.sinks) {
        const float t = a.sinks[h] * kLog2e, top = fmaxf(mx, t), base = top == neg_inf() ? 0.f : top;
        const float w = __builtin_amdgcn_exp2f(mx - base), l = ls * w + __builtin_amdgcn_exp2f(t - base);
        f = l == 0.f ? 0.f : w / l;
    } else {
        f = ls == 0.f ? 0.f : 1.f / ls;
    }
    uint16_t* const to = a.out + (size_t)(q0 + i) * a.ldo + (size_t)h * D + 4 * kg;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            *(uint2*)(to + 32 * d + 8 * e) = make_uint2(mx_bf16x2(o[d][4 * e] * f, o[d][4 * e + 1] * f), mx_bf16x2(o[d][4 * e + 2] * f, o[d][4 * e + 3] * f));
}

template <int D, int WAVES>
int launch(PromptArgs& a, hipStream_t s) {
    constexpr int kLds = 2 * 2 * kTile * 2 * D, kSize = 32 * WAVES;
    const int64_t tiles = (int64_t)a.rows / kSize + a.n;                     // a sequence's last tile may be short
    if (tiles > 0x7fffffff || !grid_fits((uint64_t)tiles * a.heads, 64 * WAVES)) return QMM_ERR_SHAPE;
    a.tiles = (int)tiles;
    hipLaunchKernelGGL((k_attn_prompt<D, WAVES>), dim3((unsigned)(tiles * a.heads)), dim3(64 * WAVES), kLds, s, a);
    QMM_LAUNCH_CHECK();
    return QMM_OK;
}

}  // namespace
}  // namespace qmm

using namespace qmm;

extern "C" int qmm_attn_prompt_bf16(const uint16_t* q, size_t ldq, const uint16_t* k, size_t ldk, const uint16_t* v, size_t ldv, uint16_t* out, size_t ldo,
                                    const int32_t* cuq, const int32_t* cuk, int nseq, const qmm_attn* attn, int rows, int krows, int heads,
                                    int kv_heads, int dim, void* stream) {
    if (dim != 64 && dim != 128 && dim != 256) return QMM_ERR_SHAPE;
    if (rows < 0 || krows < 0 || nseq < 0 || heads < 1 || kv_heads < 1 || heads > 65536 || heads % kv_heads) return QMM_ERR_SHAPE;
    if (const int st = attn_check(attn)) return st;
    if (rows == 0 || nseq == 0) return QMM_OK;
    if (!q || !out || !cuq || (krows && (!k || !v))) return QMM_ERR_NULL;
    const size_t nq = (size_t)heads * dim, nk = (size_t)kv_heads * dim;
    if (ldq < nq || ldo < nq || ldk < nk || ldv < nk || ldk > kMaxLd || ldv > kMaxLd) return QMM_ERR_SHAPE;
    if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 16) || ((ldq | ldk | ldv | ldo) & 7)) return QMM_ERR_ARG;
    if (!aligned(cuq, 4) || !aligned(cuk, 4)) return QMM_ERR_ARG;
    PromptArgs a{q, k, v, out, cuq, cuk, attn->sinks, ldq, ldo, (uint32_t)ldk, (uint32_t)ldv, 0.f, 0u,
                 nseq, attn->window, rows, krows, heads, heads / kv_heads, 0};
    // a scale of 0 (all keys weigh the same) as 2^-126: times a masked score, -inf, it is still -inf
    a.scale = fmaxf((float)(fabs((double)attn->scale) * 1.44269504088896340736), 0x1p-126f);
    a.flip = attn->scale < 0.f ? 0x80008000u : 0u;
    hipStream_t s = (hipStream_t)stream;
    switch (dim) {
        case 64: return launch<64, 4>(a, s);
        case 128: return launch<128, 4>(a, s);
        default: return launch<256, 4>(a, s);
    }
}
