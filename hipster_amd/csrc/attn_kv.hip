// attn_kv.hip -- attention of a few new rows a sequence (decode, draft verification) over a paged MXFP4 cache.
//
//   k_attn_kv     one chunk of a sequence's keys, one kv head, up to 16 NT rows (tokens x heads that share the kv head)
//   k_attn_join   a row's chunks into its output
//
// Per row: t_j = scale log2(e) q . k_j, o = sum_j 2^(t_j - m) v_j / (sum_j 2^(t_j - m) + 2^(sink log2(e) - m)), in one pass with the
// running maximum m (f32 all of it; the products' factors are bf16, see WIDE).
//
// Bound by HBM: the cache is read once, 17/16 bytes a key and value pair of one dimension, and everything else is made to fit beside it.
//   - Products run on the 16 x 16 x 32 bf16 matrix instruction with keys as rows: S^T = K Q^T, O^T = V^T P^T.  A lane of S^T holds four
//     successive keys of one query row, which is just what the second product takes of P^T from it, so P never leaves its registers.
//   - A key's codes become the first product's operand where they were loaded: lane l has 32 dims (a block: 16 bytes, one
//     scale) of key l % 16, one conversion instruction makes two bf16 of them, scale included, exactly.  Which dims a lane's eight
//     of a step are does not matter as long as Q's operand has the same.
//   - Values have to be turned (the second product sums over keys): a wave writes 32 keys' values as bf16 into LDS of its own and reads
//     them back with the transposing read, four keys of 16 dims at a time.  Rows are 32 bytes longer than their values, so that four
//     rows' 32 bytes lie in different banks.
// The four waves of a workgroup take the chunk's steps of 32 keys in turn and join their (m, l, O) through LDS in order.
//
// A chunk's length goes by max_len alone, its steps lie at fixed multiples of 32 keys, and keys that a row does not see add exact
// zeros.  So a row's bits do not depend on the other rows and sequences: a draft's rows checked together are what one by one gives.
#include "attn.hpp"

namespace qmm {
namespace {

constexpr int kWaves = 4, kStep = 32, kMaxRows = 16, kMaxShare = 16, kChunks = 128, kChunk = 256, kMaxLen = 1 << 30;

struct AttnArgs {
    const void* q;
    void* out;
    float* part;                                         // [rows * heads][chunks][D], not used with one chunk
    float* ml;                                           // [rows * heads][chunks][2]: m, l
    qmm_kv_mxfp4 kv;
    qmm_seqs s;
    const float* sinks;
    size_t ldq, ldo;
    float scale;                                         // times log2(e)
    int lg, window, rows, heads, share, max_rows, max_len, chunk, chunks, groups;   // groups: of 16 NT rows
    int q_bf, out_bf;
};

__host__ __device__ constexpr int v_stride(int D) { return 2 * D + 32; }       // bytes of a key's values in LDS

// the positions that a token at `pos` sees, [lo, hi]
struct Sight { int lo, hi; };
__device__ __forceinline__ Sight sight(const AttnArgs& a, int pos) {
    const int cap = min(a.s.ld << a.lg, a.max_len);
    return {a.window > 0 && pos >= a.window ? pos - a.window + 1 : 0, min(pos, cap - 1)};
}

__device__ __forceinline__ float max_xor16(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_xor32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_xor16(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float sum_xor32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// 2^(x - m), 0 for x = -inf whatever m
__device__ __forceinline__ float weight(float x, float m) { return __builtin_amdgcn_exp2f(x - (m == neg_inf() ? 0.f : m)); }

// o / (l + sink's weight); a row that saw nothing and has no sink: 0
__device__ __forceinline__ float finish(float o, float l, float m, const float* sinks, int h) {
    if (sinks) {
        const float t = sinks[h] * kLog2e, top = fmaxf(m, t);
        const float w = weight(m, top);
        o *= w;
        l = l * w + weight(t, top);
    }
    return l == 0.f ? 0.f : o / l;
}

__device__ __forceinline__ void put(const AttnArgs& a, size_t at, float v) {
    if (a.out_bf) ((uint16_t*)a.out)[at] = (uint16_t)mx_bf16x2(v, 0.f);
    else ((float*)a.out)[at] = v;
}

__device__ __forceinline__ uint32_t fp4x2(uint32_t code, int byte, float s) {
    at_bf2 r;
    switch (byte) {                                      // a constant after unrolling
        case 0: r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, s, 0); break;
        case 1: r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, s, 1); break;
        case 2: r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, s, 2); break;
        default: r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, s, 3);
    }
    return __builtin_bit_cast(uint32_t, r);
}
// eight values of a block
__device__ __forceinline__ uint4 fp4x8(uint32_t code, float s) { return make_uint4(fp4x2(code, 0, s), fp4x2(code, 1, s), fp4x2(code, 2, s), fp4x2(code, 3, s)); }

// The codes and scales of 16 keys as a lane has them: key l % 16; D = 64: 8 bytes, half a block; 128: a block; 256: blocks
// l / 16 and 4 + l / 16
template <int D>
struct Tile {
    static constexpr int W = D / 32;                     // words of codes = matrix steps of 32 dims
    static constexpr int S = D == 256 ? 2 : 1;           // scales
    uint32_t c[W];
    uint32_t e[S];
    __device__ __forceinline__ float scale(int w) const { return __uint_as_float(e[D == 256 ? w / 4 : 0] << 23); }
    // dim of the first of the eight values of word w, lane group kg
    static __device__ __forceinline__ int dim(int w, int kg) { return D == 64 ? kg * 16 + w * 8 : D == 128 ? kg * 32 + w * 8 : (w / 4) * 128 + kg * 32 + (w % 4) * 8; }

    __device__ __forceinline__ void load(const uint8_t* __restrict__ q, const uint8_t* __restrict__ se, size_t token, int kg) {
        const uint8_t* p = q + token * (D / 2);
        const uint8_t* s = se + token * (D / 32);
        if constexpr (D == 64) {
            const uint2 v = *(const uint2*)(p + kg * 8);
            c[0] = v.x; c[1] = v.y;
            e[0] = s[kg / 2];
        } else {
#pragma unroll
            for (int i = 0; i < S; ++i) {
                const uint4 v = *(const uint4*)(p + i * 64 + kg * 16);
                c[4 * i] = v.x; c[4 * i + 1] = v.y; c[4 * i + 2] = v.z; c[4 * i + 3] = v.w;
                e[i] = s[i * 4 + kg];
            }
        }
    }
};

template <int D>
struct Step { Tile<D> k[2], v[2]; };

// WIDE: q in f32 as three bf16 that add up to it, P as two (the second what the first's rounding missed: 2^-17 of a weight).
// Else q is bf16 and P rounded to it (2^-9 of a weight at most), as the output is.
template <int D, int NT, bool WIDE>
__global__ void __launch_bounds__(64 * kWaves) k_attn_kv(AttnArgs a) {
    constexpr int W = Tile<D>::W, QT = WIDE ? 3 : 1, DT = D / 16;
    constexpr int kVBytes = kStep * v_stride(D), kOBytes = 16 * (D + 4) * 4, kOwn = kVBytes > kOBytes ? kVBytes : kOBytes;
    __shared__ __align__(16) uint8_t lds[kWaves * kOwn];
    __shared__ float s_m[kWaves][16], s_l[kWaves][16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, kg = lane >> 4;

    const uint32_t id = blockIdx.x, chunk = id % (uint32_t)a.chunks, rest = id / (uint32_t)a.chunks;
    const uint32_t ny = (uint32_t)(a.kv.heads * a.groups), b = rest / ny, y = rest - b * ny;
    const int hk = (int)(y / (uint32_t)a.groups), group = (int)(y - hk * a.groups);

    const SeqSpan q = seq_span(a.s.cu, a.s.lens, (int)b, a.rows);
    const int m = min(q.m, a.max_rows);                  // rows of this call
    const int f0 = group * 16 * NT, fn = min(m * a.share - f0, 16 * NT);     // the group's first (token, head), and how many
    if (fn <= 0) return;
    const int first_pos = q.len - q.m;
    const int kmin = sight(a, first_pos + f0 / a.share).lo, kmax = sight(a, first_pos + (f0 + fn - 1) / a.share).hi;
    const int c0 = (int)chunk * a.chunk, c1 = min(c0 + a.chunk - 1, kmax);   // the chunk's keys, [c0, c1]; chunks * chunk < 2^31
    if (a.chunks > 1 && (c0 > kmax || c0 + a.chunk <= kmin)) return;         // the join does not look at it

    // the rows' queries as operands, and what they see
    at_bf8 qf[NT][W][QT];
    int lo[NT], hi[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int f = f0 + 16 * n + col;
        const bool live = 16 * n + col < fn;
        const int i = live ? f / a.share : 0, h = hk * a.share + (live ? f - i * a.share : 0);
        const Sight st = sight(a, first_pos + i);
        lo[n] = st.lo;
        hi[n] = live ? st.hi : -1;
        const size_t at = (size_t)(q.r0 + i) * a.ldq + (size_t)h * D;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const size_t d = at + Tile<D>::dim(w, kg);
            if constexpr (!WIDE) {
                qf[n][w][0] = *(const at_bf8*)((const uint16_t*)a.q + d);
            } else {
                float v[8];
                if (a.q_bf) {
                    const uint4 r = *(const uint4*)((const uint16_t*)a.q + d);
                    const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = __uint_as_float((j & 1) ? u[j / 2] & 0xffff0000u : u[j / 2] << 16);
                } else {
                    const float4 r0 = *(const float4*)((const float*)a.q + d), r1 = *(const float4*)((const float*)a.q + d + 4);
                    v[0] = r0.x; v[1] = r0.y; v[2] = r0.z; v[3] = r0.w; v[4] = r1.x; v[5] = r1.y; v[6] = r1.z; v[7] = r1.w;
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float left = v[j];
#pragma unroll
                    for (int t = 0; t < 3; ++t) {
                        const __bf16 p = (__bf16)left;
                        qf[n][w][t][j] = p;
                        left -= (float)p;
                    }
                    if (!(fabsf(v[j]) < 0x1.fep127f)) {  // not finite (or rounds to it): the rests would be NaN
                        qf[n][w][0][j] = (__bf16)v[j];
                        qf[n][w][1][j] = qf[n][w][2][j] = (__bf16)0.f;
                    }
                }
            }
        }
    }

    mx_v4f o[NT][DT];
    float mx[NT], ls[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        mx[n] = neg_inf();
        ls[n] = 0.f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[n][d] = mx_v4f{0.f, 0.f, 0.f, 0.f};
    }

    uint8_t* const own = lds + wave * kOwn;
    const int* const table = a.s.table + (size_t)b * a.s.ld;
    int block = -1, entry = 0;                           // lane l: the page of the 16 keys from 1024 block + 16 l on
    auto load = [&](int key0, Step<D>& st) {             // the step of the 32 keys from key0 on
        if ((key0 >> 10) != block) {
            block = key0 >> 10;
            const int pg = ((block << 10) + lane * 16) >> a.lg;
            entry = pg < a.s.ld ? table[pg] : -1;
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int k0 = key0 + 16 * t;
            int page = __builtin_amdgcn_readlane(entry, (k0 >> 4) & 63);
            const bool bad = (unsigned)page >= (unsigned)a.kv.pages;
            page = bad ? 0 : page;
            const size_t token = ((size_t)page * a.kv.heads + hk) * a.kv.page + (k0 & (a.kv.page - 1)) + col;
            st.k[t].load(a.kv.kq, a.kv.ke, token, kg);
            st.v[t].load(a.kv.vq, a.kv.ve, token, kg);
            if (bad) {                                   // scores of NaN for the rows that see these keys
#pragma unroll
                for (int i = 0; i < Tile<D>::S; ++i) st.k[t].e[i] = 255;
            }
        }
    };

    const int s0 = max((kmin - c0) & ~(kStep - 1), 0);   // kmin < c0 + chunk
    int key0 = c0 + s0 + kStep * ((wave - s0 / kStep) & (kWaves - 1));
    Step<D> cur, next;
    if (key0 <= c1) load(key0, cur);
    for (; key0 <= c1; key0 += kStep * kWaves) {
        const int after = key0 + kStep * kWaves;
        if (after <= c1) load(after, next);
        const bool inside = key0 >= kmin && key0 + kStep - 1 <= kmax;        // every key is seen by a row: none is other memory
        // values whose scale is NaN, and keys that no row sees: out of the products
        unsigned long long nan[2][Tile<D>::S];
        bool any = false;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int key = key0 + 16 * t + col;
            const bool seen = inside || (key >= kmin && key <= kmax);
#pragma unroll
            for (int i = 0; i < Tile<D>::S; ++i) {
                const bool is = cur.v[t].e[i] == 255;
                nan[t][i] = __ballot(is && seen);
                any |= nan[t][i] != 0;
                if (is || !seen) {
                    cur.v[t].e[i] = 127;
#pragma unroll
                    for (int w = 0; w < W / Tile<D>::S; ++w) cur.v[t].c[i * (W / Tile<D>::S) + w] = 0;
                }
            }
        }
        // values to LDS
        wave_fence();
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int w = 0; w < W; ++w)
                *(uint4*)(own + (16 * t + col) * v_stride(D) + 2 * Tile<D>::dim(w, kg)) = fp4x8(cur.v[t].c[w], cur.v[t].scale(w));
        // scores
        mx_v4f sc[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) sc[n][0] = sc[n][1] = mx_v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const at_bf8 kf = __builtin_bit_cast(at_bf8, fp4x8(cur.k[t].c[w], cur.k[t].scale(w)));
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int p = 0; p < QT; ++p) sc[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[n][w][p], sc[n][t], 0, 0, 0);
            }
        at_bf8 pf[NT][WIDE ? 2 : 1];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float top = neg_inf();
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = key0 + 16 * t + 4 * kg + i;
                    float v = sc[n][t][i] * a.scale;
                    if (key < lo[n] || key > hi[n]) v = neg_inf();
                    sc[n][t][i] = v;
                    top = fmaxf(top, v);
                }
            top = max_xor32(max_xor16(top));
            const float was = mx[n], now = fmaxf(was, top);
            if (__ballot(now != was)) {                  // times 1 where it is the same
                const float f = weight(was, now);
                ls[n] *= f;
#pragma unroll
                for (int d = 0; d < DT; ++d) o[n][d] *= f;
                mx[n] = now;
            }
            const float base = now == neg_inf() ? 0.f : now;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p = __builtin_amdgcn_exp2f(sc[n][t][i] - base);
                    ls[n] += p;
                    const __bf16 r = (__bf16)p;
                    pf[n][0][4 * t + i] = r;
                    if constexpr (WIDE) pf[n][1][4 * t + i] = (__bf16)(p - (float)r);
                }
        }
        wave_fence();                                    // other lanes read what this one wrote
        // values by transposing reads: lane l gets dim 16 d + l % 16 of the keys 16 t + 4 kg .. + 3
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const uint8_t* from = own + (4 * kg + (col >> 2)) * v_stride(D) + 32 * d + 8 * (col & 3);
            const at_s4 v0 = tr_read(from), v1 = tr_read(from + 16 * v_stride(D));
            const at_bf8 vf = __builtin_bit_cast(at_bf8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int p = 0; p < (WIDE ? 2 : 1); ++p) o[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[n][p], o[n][d], 0, 0, 0);
        }
        if (any) {                                       // uniform, and rare: a key's block of NaN reaches the rows that see the key
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < Tile<D>::S; ++i)
                    for (unsigned long long left = nan[t][i]; left; left &= left - 1) {
                        const int l = __builtin_ctzll(left), key = key0 + 16 * t + (l & 15);
                        const int blk = D == 64 ? (l >> 4) / 2 : i * 4 + (l >> 4);
#pragma unroll
                        for (int n = 0; n < NT; ++n)
                            if (key >= lo[n] && key <= hi[n]) {
#pragma unroll
                                for (int d = 0; d < DT; ++d)
                                    if (d / 2 == blk) o[n][d] = mx_v4f{1.f, 1.f, 1.f, 1.f} * __uint_as_float(0x7fc00000u);
                            }
                    }
        }
        cur = next;
    }

    // the four waves' sums in order; lane (col, kg) has dims 16 d + 4 kg .. + 3 of row col
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        __syncthreads();                                 // the values, or the rows before, are read
        float* const mine = (float*)own;
#pragma unroll
        for (int d = 0; d < DT; ++d) *(mx_v4f*)(mine + col * (D + 4) + 16 * d + 4 * kg) = o[n][d];
        const float l = sum_xor32(sum_xor16(ls[n]));
        if (kg == 0) { s_m[wave][col] = mx[n]; s_l[wave][col] = l; }
        __syncthreads();
        for (int at = threadIdx.x; at < 16 * D; at += 64 * kWaves) {
            const int r = at / D, d = at % D;
            if (16 * n + r >= fn) continue;
            float top = s_m[0][r];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) top = fmaxf(top, s_m[w][r]);
            float v = 0.f, sum = 0.f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float f = weight(s_m[w][r], top);
                v += f * ((const float*)(lds + w * kOwn))[r * (D + 4) + d];
                sum += f * s_l[w][r];
            }
            const int f = f0 + 16 * n + r, i = f / a.share, h = hk * a.share + f - i * a.share;
            const size_t row = (size_t)(q.r0 + i);
            if (a.chunks == 1) {
                put(a, row * a.ldo + (size_t)h * D + d, finish(v, sum, top, a.sinks, h));
            } else {
                const size_t to = (row * a.heads + h) * a.chunks + chunk;
                a.part[to * D + d] = v;
                if (d == 0) { a.ml[2 * to] = top; a.ml[2 * to + 1] = sum; }
            }
        }
    }
}

// One workgroup per row and head: its chunks' weights, then D values as groups of threads that take the chunks in turn, joined in order.
template <int D>
__global__ void __launch_bounds__(256) k_attn_join(AttnArgs a) {
    constexpr int L = D / 4, G = 256 / L;                // lanes of a group, groups
    __shared__ float s_w[kChunks], s_red[8];
    __shared__ __align__(16) float s_o[G][D];
    const int tid = threadIdx.x, wave = tid >> 6;
    const uint32_t row = blockIdx.x / (uint32_t)a.heads, h = blockIdx.x - row * a.heads;
    const int b = seq_of_row(a.s.cu, a.s.n, (int)row);
    if (b < 0) return;
    const SeqSpan q = seq_span(a.s.cu, a.s.lens, b, a.rows);
    const int i = (int)row - q.r0;
    if (i < 0 || i >= min(q.m, a.max_rows)) return;
    const Sight st = sight(a, q.len - q.m + i);
    const size_t to = (size_t)row * a.ldo + (size_t)h * D, at = ((size_t)row * a.heads + h) * a.chunks;
    const int first = st.lo / a.chunk, last = st.hi < st.lo ? -1 : st.hi / a.chunk;              // its chunks, below kChunks
    const bool live = tid >= first && tid <= last;
    float m = neg_inf(), l = 0.f;
    if (live) { m = a.ml[2 * (at + tid)]; l = a.ml[2 * (at + tid) + 1]; }
    float top = m;
    for (int k = 32; k; k >>= 1) top = fmaxf(top, __shfl_xor(top, k, 64));
    if ((tid & 63) == 0) s_red[wave] = top;
    __syncthreads();
    top = fmaxf(s_red[0], s_red[1]);                     // two waves have all the chunks
    const float w = live ? weight(m, top) : 0.f;
    if (tid < kChunks) s_w[tid] = w;
    const float sum = wave_sum(w * l);                   // a chunk's place in the sums goes by its number alone
    if ((tid & 63) == 0) s_red[4 + wave] = sum;
    __syncthreads();
    const int g = tid / L, d = (tid % L) * 4;
    mx_v4f o = {0.f, 0.f, 0.f, 0.f};
    for (int c = first - first % G + g; c <= last; c += G)
        if (c >= first) o += s_w[c] * *(const mx_v4f*)(a.part + (at + c) * D + d);
    *(mx_v4f*)&s_o[g][d] = o;
    __syncthreads();
    if (tid < D) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < G; ++k) v += s_o[k][tid];
        put(a, to + tid, finish(v, s_red[4] + s_red[5], top, a.sinks, (int)h));
    }
}

// keys of a chunk: 256, or as many as make 128 chunks of max_len
int chunk_of(int max_len) {
    int c = kChunk;
    while ((int64_t)c * kChunks < max_len) c *= 2;
    return c;
}
int chunks_of(int max_len) { return (max_len + chunk_of(max_len) - 1) / chunk_of(max_len); }

template <int D, int NT, bool WIDE>
int launch(AttnArgs& a, hipStream_t s) {
    a.groups = (a.max_rows * a.share + 16 * NT - 1) / (16 * NT);
    const uint64_t grid = (uint64_t)a.s.n * a.kv.heads * a.groups * a.chunks;
    if (!grid_fits(grid, 64 * kWaves) || !grid_fits((uint64_t)a.rows * a.heads, 256)) return QMM_ERR_SHAPE;
    hipLaunchKernelGGL((k_attn_kv<D, NT, WIDE>), dim3((unsigned)grid), dim3(64 * kWaves), 0, s, a);
    QMM_LAUNCH_CHECK();
    if (a.chunks > 1) {
        hipLaunchKernelGGL((k_attn_join<D>), dim3((unsigned)(a.rows * a.heads)), dim3(256), 0, s, a);
        QMM_LAUNCH_CHECK();
    }
    return QMM_OK;
}

// rows of a workgroup: 16, 32 or 64, what covers a sequence's; fewer where operands and sums would not fit 256 registers
template <int D>
int launch_rows(AttnArgs& a, bool wide, hipStream_t s) {
    const int f = a.max_rows * a.share;
    if (wide) {
        if (f <= 16 || D == 256) return launch<D, 1, true>(a, s);
        if constexpr (D < 256) return launch<D, 2, true>(a, s);
    }
    if (f <= 16) return launch<D, 1, false>(a, s);
    if (f <= 32 || D == 256) return launch<D, 2, false>(a, s);
    if constexpr (D < 256) return launch<D, 4, false>(a, s);
    return QMM_ERR_SHAPE;                                // not reached
}

}  // namespace
}  // namespace qmm

using namespace qmm;

extern "C" {

size_t qmm_attn_kv_ws_bytes(int rows, int heads, int dim, int max_len) {
    if (rows <= 0 || heads <= 0 || max_len <= 0 || max_len > kMaxLen || (dim != 64 && dim != 128 && dim != 256)) return 0;
    const int n = chunks_of(max_len);
    return n == 1 ? 0 : (size_t)rows * heads * n * (dim + 2) * sizeof(float);
}

int qmm_attn_kv_mxfp4(const void* q, int q_dtype, size_t ldq, const qmm_kv_mxfp4* kv, const qmm_seqs* seqs, const qmm_attn* attn, void* out,
                      int out_dtype, size_t ldo, int rows, int heads, int max_rows, int max_len, void* ws, size_t ws_bytes, void* stream) {
    if ((q_dtype != QMM_F32 && q_dtype != QMM_BF16) || (out_dtype != QMM_F32 && out_dtype != QMM_BF16)) return QMM_ERR_FORMAT;
    if (rows < 0) return QMM_ERR_SHAPE;
    if (rows == 0) return QMM_OK;
    if (!q || !out) return QMM_ERR_NULL;
    AttnArgs a;
    if (const int st = kv_check(kv, seqs, &a.lg)) return st;
    if (const int st = attn_check(attn)) return st;
    if (heads < 1 || heads % kv->heads || heads / kv->heads > kMaxShare || max_rows < 1 || max_rows > kMaxRows || max_len < 1 || max_len > kMaxLen) return QMM_ERR_SHAPE;
    const size_t n = (size_t)heads * kv->dim;
    if (ldq < n || ldo < n) return QMM_ERR_SHAPE;
    const bool qb = q_dtype == QMM_BF16, ob = out_dtype == QMM_BF16;
    if (!aligned(q, 16) || ldq % (qb ? 8 : 4) || !aligned(out, ob ? 2 : 4)) return QMM_ERR_ARG;
    const size_t need = qmm_attn_kv_ws_bytes(rows, heads, kv->dim, max_len);
    if (need && (!ws || ws_bytes < need)) return QMM_ERR_WORKSPACE;
    if (need && !aligned(ws, 16)) return QMM_ERR_ARG;
    a.q = q; a.out = out; a.kv = *kv; a.s = *seqs; a.sinks = attn->sinks; a.ldq = ldq; a.ldo = ldo;
    a.scale = (float)((double)attn->scale * 1.44269504088896340736);
    a.window = attn->window; a.rows = rows; a.heads = heads; a.share = heads / kv->heads; a.max_rows = max_rows; a.max_len = max_len;
    a.chunk = chunk_of(max_len);
    a.chunks = chunks_of(max_len);
    a.part = (float*)ws;
    a.ml = a.part + (need ? (size_t)rows * heads * a.chunks * kv->dim : 0);
    a.q_bf = qb; a.out_bf = ob;
    hipStream_t s = (hipStream_t)stream;
    const bool wide = !qb || !ob;
    switch (kv->dim) {
        case 64: return launch_rows<64>(a, wide, s);
        case 128: return launch_rows<128>(a, wide, s);
        default: return launch_rows<256>(a, wide, s);
    }
}

}  // extern "C"
