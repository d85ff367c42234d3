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
//     them back with the transposing read, four keys of 16 dims at a time.
// The waves of a workgroup take the chunk's steps of 32 keys in turn and join their (m, l, O) through LDS in order.
//
// 32 heads on 8 of 128 dims, 32 sequences of up to 8192 keys, 180 MB: 50 us with the join's 4.8 on caches in turn, 45 on one again and again, which
// the last-level cache holds (as in all the times below; loads alone then 34 and the join).  700 keys of one sequence 9.2 us.
// The join of a workgroup's waves after each chunk, with the sums it writes, takes 5.5 of these us (44.4 traced, without it 38.9), and 8.3 of 44.0 where 16
// such sequences check 8 drafted rows each, 64 heads on 8 of 64 dims.  The larger part there is vector instructions: 387 of a wave for 32
// keys and 64 rows (codes 40, the rest the softmax of four groups of rows) and 88 of the waves' join, 59 % of a SIMD's cycles with two waves on it.
//
// A chunk's length goes by max_len and the dims alone, its steps lie at fixed multiples of 32 keys, and keys that a row does not see add exact
// zeros.  So a row's bits do not depend on the other rows and sequences: a draft's rows checked together are what one by one gives.
#include "attn.hpp"

#include <algorithm>

namespace qmm {
namespace {

constexpr int kStep = 32, kMaxRows = 16, kMaxShare = 16, kChunks = 128, kMaxLen = 1 << 30, kNone = 0x7fff0000;
constexpr float kSlack = 8.f;

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
    int lgc;                                             // log2 of chunk
    int q_bf, out_bf, out_vec;                           // out_vec: four values of a row of out are aligned
};

// A key's values in LDS: 2 D bytes, its 16-byte piece p at p ^ v_turn(key).  What is written together (a piece of eight keys) and read
// together (two pieces of eight keys) then lies in different banks.
template <int D>
__device__ __forceinline__ uint32_t v_turn(int key) { return (uint32_t)(D == 64 ? key & 7 : (key & 7) ^ ((key & 1) << 3)); }

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

// The units of work, in order: sequence, kv head, group of 16 NT rows, chunk.  What a call has of them is known on the device alone;
// each workgroup counts them and takes its share.  A unit's place: its sequence, that one's chunks (from `first` on) and groups, and
// the unit's number in it (`units`); past the last unit: `units` is how many there are.  The wave adds up 64 sequences at a time.
struct Place { int b, first, chunks, groups; uint32_t units; SeqSpan q; };
struct Counts { int first, chunks, groups; uint32_t mine, upto; SeqSpan q; };           // a lane's sequence; upto: of the sequences to it

template <int NT>
__device__ __forceinline__ Counts count(const AttnArgs& a, int base) {
    const int lane = threadIdx.x & 63;
    Counts c = {0, 0, 0, 0, 0, {0, 0, 0}};
    if (base + lane < a.s.n) {
        const SeqSpan q = c.q = seq_span(a.s.cu, a.s.lens, base + lane, a.rows);
        const int m = min(q.m, a.max_rows);
        if (m > 0) {
            const int lo = sight(a, q.len - q.m).lo, hi = sight(a, q.len - q.m + m - 1).hi;
            c.first = a.chunks == 1 ? 0 : lo >> a.lgc;
            c.chunks = a.chunks == 1 ? 1 : hi < lo ? 0 : (hi >> a.lgc) - c.first + 1;
            c.groups = (m * a.share + 16 * NT - 1) / (16 * NT);
        }
    }
    c.mine = (uint32_t)(c.chunks * c.groups * a.kv.heads);
    c.upto = wave_upto(c.mine);
    return c;
}
// the place of a unit that lies in the 64 sequences counted in c, `before` units lying in front of them
__device__ __forceinline__ bool pick(const Counts& c, int base, uint32_t before, uint32_t unit, Place& p) {
    const unsigned long long behind = __ballot(before + c.upto > unit);
    if (!behind) return false;
    const int l = __builtin_ctzll(behind);
    p = {base + l, __builtin_amdgcn_readlane(c.first, l), __builtin_amdgcn_readlane(c.chunks, l), __builtin_amdgcn_readlane(c.groups, l),
         unit - before - (uint32_t)__builtin_amdgcn_readlane((int)(c.upto - c.mine), l),
         {__builtin_amdgcn_readlane(c.q.r0, l), __builtin_amdgcn_readlane(c.q.m, l), __builtin_amdgcn_readlane(c.q.len, l)}};
    return true;
}
template <int NT>
__device__ __forceinline__ Place locate(const AttnArgs& a, uint32_t unit) {
    Place p = {-1, 0, 1, 1, 0, {0, 0, 0}};
    for (int base = 0; base < a.s.n; base += 64) {
        const Counts c = count<NT>(a, base);
        if (pick(c, base, p.units, unit, p)) return p;
        p.units += (uint32_t)__builtin_amdgcn_readlane((int)c.upto, 63);
    }
    return p;
}
// the workgroup's first unit and the one after its last, and the first one's place: as many as any other's, one more at most
template <int NT>
__device__ __forceinline__ Place share(const AttnArgs& a, uint32_t& unit, uint32_t& end) {
    Place p = {-1, 0, 1, 1, 0, {0, 0, 0}};
    const bool once = a.s.n <= 64;
    Counts c;
    if (once) c = count<NT>(a, 0);
    const uint64_t total = once ? (uint32_t)__builtin_amdgcn_readlane((int)c.upto, 63) : locate<NT>(a, 0xffffffffu).units;
    unit = (uint32_t)(total * blockIdx.x / gridDim.x);
    end = (uint32_t)(total * (blockIdx.x + 1) / gridDim.x);
    if (unit < end) {
        if (once) pick(c, 0, 0, unit, p);
        else p = locate<NT>(a, unit);
    }
    return p;
}

// four values of a row
__device__ __forceinline__ void put4(const AttnArgs& a, size_t at, const mx_v4f& v) {
    if (a.out_bf) mx_store4<true>(a.out, at, v, 4, a.out_vec);
    else mx_store4<false>(a.out, at, v, 4, a.out_vec);
}

// v, an f32, as three bf16 that add up to it: its leading 8 significant bits, the next 8 and the last 8 (dropping bits, not rounding,
// keeps each rest exact and costs one instruction).  Not finite: the first alone.
__device__ __forceinline__ void split3(const float (&v)[8], at_bf8 (&f)[3]) {
    uint32_t w[3][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t x[2][3];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t u = __float_as_uint(v[2 * j + i]);
            const float a = __uint_as_float(u & 0xffff0000u), r = v[2 * j + i] - a, b = __uint_as_float(__float_as_uint(r) & 0xffff0000u);
            x[i][0] = u;
            x[i][1] = __float_as_uint(r);
            x[i][2] = __float_as_uint(r - b);
        }
#pragma unroll
        for (int t = 0; t < 3; ++t) w[t][j] = __builtin_amdgcn_perm(x[1][t], x[0][t], 0x07060302u);      // the upper halves
    }
#pragma unroll
    for (int t = 0; t < 3; ++t) f[t] = __builtin_bit_cast(at_bf8, make_uint4(w[t][0], w[t][1], w[t][2], w[t][3]));
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
    static constexpr int V = W / S;                      // words of a load
    typedef uint32_t Codes __attribute__((ext_vector_type(V)));
    Codes c[S];
    uint32_t e[S];
    __device__ __forceinline__ uint32_t word(int w) const { return c[w / V][w % V]; }
    __device__ __forceinline__ float scale(int w) const { return __uint_as_float(e[w / V] << 23); }
    __device__ __forceinline__ void nan_out() {          // what counts as NaN to NaN
#pragma unroll
        for (int i = 0; i < S; ++i) e[i] = e[i] >= kMxNan ? 255 : e[i];
    }
    __device__ __forceinline__ void clear(int i) {       // to values of 0
        c[i] = Codes(0);
        e[i] = 127;
    }
    // dim of the first of the eight values of word w, lane group kg
    static __device__ __forceinline__ int dim(int w, int kg) { return D == 64 ? kg * 16 + w * 8 : D == 128 ? kg * 32 + w * 8 : (w / 4) * 128 + kg * 32 + (w % 4) * 8; }

    __device__ __forceinline__ void load(const uint8_t* __restrict__ q, const uint8_t* __restrict__ se, size_t token, int kg) {
        const uint8_t* p = q + token * (D / 2);
        const uint8_t* s = se + (D == 64 ? token & ~(size_t)1 : token) * (D / 32);        // D = 64: a word is two keys' bytes
#pragma unroll
        for (int i = 0; i < S; ++i) {
            c[i] = *(const Codes*)(p + i * 64 + kg * (4 * V));
            e[i] = *(const uint32_t*)(s + 4 * i);
        }
    }
    // to the lane's scale bytes from the words that hold them
    __device__ __forceinline__ void open(int shift) {
#pragma unroll
        for (int i = 0; i < S; ++i) e[i] = __builtin_amdgcn_ubfe(e[i], (uint32_t)shift, 8);
    }
    static __device__ __forceinline__ int shift(int col, int kg) { return D == 64 ? 16 * (col & 1) + 8 * (kg / 2) : 8 * kg; }
};

// workgroups of a CU (waves of a SIMD) that the registers are cut for
__host__ __device__ constexpr int occupancy(int D, int NT, bool wide) {
    return D == 64 ? (NT == 1 ? 4 : NT == 2 && !wide ? 3 : 2) : D == 128 ? (NT == 1 ? (wide ? 2 : 3) : NT == 2 && !wide ? 2 : 1) : NT == 1 && !wide ? 2 : 1;
}

template <int D>
struct Step { Tile<D> k[2], v[2]; bool bad[2]; };      // bad: on a page outside the cache

// WIDE: q in f32 as three bf16 that add up to it, P as three too.
// Else q is bf16 and P rounded to it (2^-8 of a weight at most), as the output is.
template <int D, int NT, bool WIDE, int NW>
__global__ void __launch_bounds__(64 * NW, occupancy(D, NT, WIDE) * 4 / NW * (NW / 4)) k_attn_kv(AttnArgs a) {
    constexpr int W = Tile<D>::W, QT = WIDE ? 3 : 1, DT = D / 16;
    constexpr int kOwn = (16 * (D + 4) * 4 + 511) / 512 * 512;               // of a wave: 32 keys' values, or 16 rows' sums
    static_assert(kOwn >= kStep * 2 * D, "");
    __shared__ __align__(512) uint8_t lds[NW * kOwn];
    __shared__ float s_m[NW][16], s_l[NW][16];
    __shared__ int s_row[16 * NT], s_head[16 * NT];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, kg = lane >> 4;

    uint32_t unit, end;
    for (Place at_unit = share<NT>(a, unit, end); unit < end;) {
    const int b = at_unit.b;
    const uint32_t y = at_unit.units / (uint32_t)at_unit.chunks;
    const int c_off = (int)(at_unit.units - y * at_unit.chunks);
    const int hk = (int)(y / (uint32_t)at_unit.groups), group = (int)(y - hk * at_unit.groups);
    const int c_end = min(at_unit.chunks - c_off, (int)(end - unit));        // units of this group here
    unit += (uint32_t)c_end;
    const int c_first = at_unit.first + c_off;
    const SeqSpan q = at_unit.q;
    if (unit < end) at_unit = locate<NT>(a, unit);       // the next group's

    const int m = min(q.m, a.max_rows);                  // rows of this call
    const int f0 = group * 16 * NT, fn = min(m * a.share - f0, 16 * NT);     // the group's first (token, head), and how many
    const int first_pos = q.len - q.m;
    const int kmin = sight(a, first_pos + f0 / a.share).lo, kmax = sight(a, first_pos + (f0 + fn - 1) / a.share).hi;
    const int lmax = sight(a, first_pos + (f0 + fn - 1) / a.share).lo, hmin = sight(a, first_pos + f0 / a.share).hi;
    // its chunks that a row of the group sees (the join looks at no other); without a join there is one, which answers for all rows
    const bool one = a.chunks == 1;
    const int cfirst = max(c_first, one ? 0 : kmin >> a.lgc);
    const int clast = min(c_first + c_end - 1, one ? 0 : kmax < 0 ? -1 : kmax >> a.lgc);
    if (cfirst > clast) continue;

    if (threadIdx.x < 16 * NT) {                         // read behind the chunks' barriers
        const int f = f0 + (int)threadIdx.x, i = f / a.share;
        s_row[threadIdx.x] = q.r0 + i;
        s_head[threadIdx.x] = hk * a.share + f - i * a.share;
    }
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
                bool odd = false;                        // infinities and NaN have rests of NaN: kept out of the sum
#pragma unroll
                for (int j = 0; j < 8; ++j) odd |= !(fabsf(v[j]) < __uint_as_float(0x7f800000u));
                at_bf8 f3[3];
                split3(v, f3);
                if (odd) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const bool is = !(fabsf(v[j]) < __uint_as_float(0x7f800000u));
                        f3[0][j] = is ? (__bf16)v[j] : f3[0][j];
                        f3[1][j] = is ? (__bf16)0.f : f3[1][j];
                        f3[2][j] = is ? (__bf16)0.f : f3[2][j];
                    }
                }
#pragma unroll
                for (int x = 0; x < QT; ++x) qf[n][w][x] = f3[x];
            }
        }
    }

    mx_v4f o[NT][DT];
    float mx[NT], ls[NT];

    uint8_t* const own = lds + wave * kOwn;
    // where this lane writes the first piece of its key's values, and where it reads those of its row (offsets below 2 D come by xor)
    const uint32_t v_to = (uint32_t)col * (2 * D) + ((uint32_t)(Tile<D>::dim(0, kg) / 8) ^ v_turn<D>(col)) * 16;
    const int v_row = 4 * kg + (col >> 2);
    const uint32_t v_from = (uint32_t)v_row * (2 * D) + ((uint32_t)((col >> 1) & 1) ^ v_turn<D>(v_row)) * 16 + 8 * (col & 1);
    const int* const table = a.s.table + (size_t)b * a.s.ld;
    int block = -1, entry = 0;                           // lane l: the page of the 16 keys from 1024 block + 16 l on
    auto wanted = [&](int key0) { return key0 <= kmax && key0 + kStep > kmin; };
    auto load = [&](int key0, Step<D>& st) {             // the step of the 32 keys from key0 on
        if ((key0 >> 10) != block) {
            block = key0 >> 10;
            const int pg = ((block << 10) + lane * 16) >> a.lg;
            entry = -1;
            if (pg < a.s.ld) entry = table[pg];
            entry = (int)opaque((uint32_t)entry);        // waited for here, not at each of its uses
        }
        size_t token[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int k0 = key0 + 16 * t;
            int page = __builtin_amdgcn_readlane(entry, (k0 >> 4) & 63);
            const bool bad = (unsigned)page >= (unsigned)a.kv.pages;
            page = bad ? 0 : page;
            token[t] = ((size_t)page * a.kv.heads + hk) * a.kv.page + (k0 & (a.kv.page - 1)) + col;
            st.bad[t] = bad;
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) st.v[t].load(a.kv.vq, a.kv.ve, token[t], kg);
#pragma unroll
        for (int t = 0; t < 2; ++t) st.k[t].load(a.kv.kq, a.kv.ke, token[t], kg);
    };

    // Steps go round the waves; of a block of 256 keys a wave has two, each with a buffer of its own, which is filled again for the next
    // block as soon as its codes are converted: two steps are under way.  A buffer is filled in one place, with words (a byte's extension is
    // work on it), and the pages' load is waited for where it is made, so that no wait of the compiler's is for the other buffer too (16
    // sequences of up to 32000 keys 111 -> 107 us).
    constexpr int kBlock = 2 * kStep * NW;
    const int blocks = a.chunk / kBlock;                 // of a chunk
    const int b0 = max(cfirst * blocks, kmin / kBlock), b1 = kmax < 0 ? -1 : min((clast + 1) * blocks - 1, kmax / kBlock);
    auto step = [&](int key0, Step<D>& st, int after) {
        const bool inside = key0 >= kmin && key0 + kStep - 1 <= kmax;        // every key is seen by a row: none is other memory
        const bool all = key0 >= lmax && key0 + kStep - 1 <= hmin;           // every row sees every key
        // values whose scale is NaN, and keys that no row sees: out of the products
        unsigned long long nan[2][Tile<D>::S], any = 0;
        const bool want = wanted(key0);
        mx_v4f sc[NT][2];
        if (want) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            st.v[t].open(Tile<D>::shift(col, kg));
            st.k[t].open(Tile<D>::shift(col, kg));
            if (!inside) {
                const int key = key0 + 16 * t + col;
                if (key < kmin || key > kmax) {
#pragma unroll
                    for (int i = 0; i < Tile<D>::S; ++i) st.v[t].clear(i);
                }
            }
#pragma unroll
            for (int i = 0; i < Tile<D>::S; ++i) {
                nan[t][i] = __ballot(st.v[t].e[i] >= kMxNan);
                any |= nan[t][i];
            }
        }
        if (any) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < Tile<D>::S; ++i)
                    if (st.v[t].e[i] >= kMxNan) st.v[t].clear(i);
        }
        st.k[0].nan_out();
        st.k[1].nan_out();
        if (st.bad[0] || st.bad[1]) {                    // scores of NaN for the rows that see these keys
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < Tile<D>::S; ++i)
                    if (st.bad[t]) st.k[t].e[i] = 255;
        }
        // values to LDS
        wave_fence();
        const uint32_t to = opaque(v_to);                // the pieces' addresses are made anew each time, not kept
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int w = 0; w < W; ++w)
                *(uint4*)(own + 16 * t * (2 * D) + (to ^ (Tile<D>::dim(w, 0) * 2))) = fp4x8(st.v[t].word(w), st.v[t].scale(w));
        // scores
#pragma unroll
        for (int n = 0; n < NT; ++n) sc[n][0] = sc[n][1] = mx_v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const at_bf8 kf = __builtin_bit_cast(at_bf8, fp4x8(st.k[t].word(w), st.k[t].scale(w)));
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int p = 0; p < QT; ++p) sc[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[n][w][p], sc[n][t], 0, 0, 0);
            }
        }
        if (wanted(after)) load(after, st);
        if (!want) return;
        at_bf8 pf[NT][QT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float top = neg_inf();
            if (all) {
#pragma unroll
                for (int t = 0; t < 2; ++t) sc[n][t] *= a.scale;
            } else {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int key = key0 + 16 * t + 4 * kg + i;
                        sc[n][t][i] = key < lo[n] || key > hi[n] ? neg_inf() : sc[n][t][i] * a.scale;
                    }
            }
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) top = fmaxf(top, sc[n][t][i]);
            top = max_xor32(max_xor16(top));
            // a row's sums go on at a new maximum only when it is past the old one by a factor of 2^8 (weights stay below that, as exact)
            const float was = mx[n], now = top > was + kSlack ? top : was;
            if (__ballot(now != was)) {                  // times 1 where it is the same
                const float f = weight(was, now);
                ls[n] *= f;
#pragma unroll
                for (int d = 0; d < DT; ++d) o[n][d] *= f;
                mx[n] = now;
            }
            const float base = now == neg_inf() ? 0.f : now;
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                p[i] = __builtin_amdgcn_exp2f(sc[n][i / 4][i % 4] - base);
                ls[n] += p[i];
            }
            if constexpr (WIDE) split3(p, pf[n]);
            else pf[n][0] = __builtin_bit_cast(at_bf8, make_uint4(mx_bf16x2(p[0], p[1]), mx_bf16x2(p[2], p[3]), mx_bf16x2(p[4], p[5]), mx_bf16x2(p[6], p[7])));
        }
        wave_fence();                                    // other lanes read what this one wrote
        // values by transposing reads: lane l gets dim 16 d + l % 16 of the keys 16 t + 4 kg .. + 3
        const uint32_t at_row = opaque(v_from);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const uint8_t* from = own + (at_row ^ (32 * d));
            const at_s4 v0 = tr_read(from), v1 = tr_read(from + 16 * 2 * D);
            const at_bf8 vf = __builtin_bit_cast(at_bf8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int p = 0; p < QT; ++p) o[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[n][p], o[n][d], 0, 0, 0);
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
                        for (int n = 0; n < NT; ++n) {
                            const float f = key >= lo[n] && key <= hi[n] ? __uint_as_float(0x7fc00000u) : 1.f;
#pragma unroll
                            for (int d = 0; d < DT; ++d) o[n][d] *= d / 2 == blk ? f : 1.f;
                        }
                    }
        }
    };

    Step<D> even, odd;
    const int own0 = kStep * wave, own1 = own0 + kStep * NW;             // its steps of a block
    if (wanted(b0 * kBlock + own0)) load(b0 * kBlock + own0, even);
    if (wanted(b0 * kBlock + own1)) load(b0 * kBlock + own1, odd);
    for (int chunk = cfirst, blk = b0; chunk <= clast; ++chunk) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        mx[n] = neg_inf();
        ls[n] = 0.f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[n][d] = mx_v4f{0.f, 0.f, 0.f, 0.f};
    }
    for (const int end = min((chunk + 1) * blocks - 1, b1); blk <= end; ++blk) {
        const int k0 = blk * kBlock, next = blk < b1 ? k0 + kBlock : kNone;
        step(k0 + own0, even, next + own0);
        step(k0 + own1, odd, next + own1);
    }

    // the waves' sums in order; lane (col, kg) has dims 16 d + 4 kg .. + 3 of row col
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        lds_barrier();                                   // the values, or the rows before, are read
        float* const mine = (float*)own;
#pragma unroll
        for (int d = 0; d < DT; ++d) *(mx_v4f*)(mine + col * (D + 4) + 16 * d + 4 * kg) = o[n][d];
        const float l = sum_xor32(sum_xor16(ls[n]));
        if (kg == 0) { s_m[wave][col] = mx[n]; s_l[wave][col] = l; }
        lds_barrier();
        const int tid = (int)opaque(threadIdx.x);        // addresses made here, not kept through the steps
#pragma unroll 1
        for (int k = 0; k < (4 * D + 64 * NW - 1) / (64 * NW); ++k) {         // four dims a thread
            const int at = tid + 64 * NW * k, r = at / (D / 4), d = at % (D / 4) * 4;
            if (r >= 16 || 16 * n + r >= fn) break;
            float top = s_m[0][r];
#pragma unroll
            for (int w = 1; w < NW; ++w) top = fmaxf(top, s_m[w][r]);
            mx_v4f v = {0.f, 0.f, 0.f, 0.f};
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float f = weight(s_m[w][r], top);
                v += f * *(const mx_v4f*)((const float*)(lds + w * kOwn) + r * (D + 4) + d);
                sum += f * s_l[w][r];
            }
            const int h = s_head[16 * n + r];
            const size_t row = (size_t)s_row[16 * n + r];
            if (a.chunks == 1) {
                const float f = finish(1.f, sum, top, a.sinks, h);
                put4(a, row * a.ldo + (size_t)h * D + d, v * f);
            } else {
                const size_t to = (row * a.heads + h) * a.chunks + chunk;
                *(mx_v4f*)(a.part + to * D + d) = v;
                if (d == 0) *(float2*)(a.ml + 2 * to) = make_float2(top, sum);
            }
        }
    }
    lds_barrier();                                       // before the next chunk's values
    }
    }
}

// One wave per row, head and 64 dims: the chunks' weights, then the dims' sums by four groups of 16 lanes that take the chunks in turn.
// A chunk's place in every sum goes by its number alone.
template <int D>
__global__ void __launch_bounds__(64) k_attn_join(AttnArgs a) {
    constexpr int P = D / 64, G = 4;                     // parts of a row's head; groups
    __shared__ float s_w[kChunks];
    const int lane = threadIdx.x;
    const uint32_t rh = blockIdx.x / P, part = blockIdx.x % P, row = rh / (uint32_t)a.heads, h = rh - row * a.heads;
    SeqSpan q;
    if (seq_of_row(a.s.cu, a.s.lens, a.s.n, a.rows, (int)row, q) < 0) return;
    const int i = (int)row - q.r0;
    if (i < 0 || i >= min(q.m, a.max_rows)) return;
    const Sight st = sight(a, q.len - q.m + i);
    const size_t at = ((size_t)row * a.heads + h) * a.chunks;
    const int first = st.lo >> a.lgc, last = st.hi < st.lo ? -1 : st.hi >> a.lgc;                // its chunks, below kChunks
    float m[kChunks / 64], l[kChunks / 64], top = neg_inf(), sum = 0.f;
#pragma unroll
    for (int k = 0; k < kChunks / 64; ++k) {
        const int c = 64 * k + lane;
        const bool live = c >= first && c <= last;
        const float2 v = live ? *(const float2*)(a.ml + 2 * (at + c)) : make_float2(neg_inf(), 0.f);
        m[k] = v.x;
        l[k] = v.y;
        top = fmaxf(top, m[k]);
    }
    for (int k = 32; k; k >>= 1) top = fmaxf(top, __shfl_xor(top, k, 64));
#pragma unroll
    for (int k = 0; k < kChunks / 64; ++k) {
        const float w = weight(m[k], top);
        s_w[64 * k + lane] = w;
        sum += w * l[k];
    }
    sum = wave_sum(sum);
    wave_fence();
    const int g = lane >> 4, d = (lane & 15) * 4;
    const float* from = a.part + at * D + part * 64 + d;
    mx_v4f o = {0.f, 0.f, 0.f, 0.f};
    for (int c0 = first & ~(8 * G - 1); c0 <= last; c0 += 8 * G) {           // eight chunks a lane asked for together
        mx_v4f v[8];
#pragma unroll
        for (int i8 = 0; i8 < 8; ++i8) {
            const int c = c0 + G * i8 + g;
            v[i8] = c >= first && c <= last ? *(const mx_v4f*)(from + (size_t)c * D) : mx_v4f{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int i8 = 0; i8 < 8; ++i8) {
            const int c = c0 + G * i8 + g;
            o += (c >= first && c <= last ? s_w[c] : 0.f) * v[i8];
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = sum_xor32(sum_xor16(o[e]));
    const float f = finish(1.f, sum, top, a.sinks, (int)h);
    if (g == 0) put4(a, (size_t)row * a.ldo + (size_t)h * D + part * 64 + d, o * f);
}

// Keys of a chunk, a power of two.  Up to 1024 keys are one chunk, which needs no join (700 keys of one sequence: 9.2 µs, as three chunks of
// 256 9.9).  Beyond, short chunks spread few sequences over the device and long ones have less to join; in µs with chunks of 256, 512, 1024:
//   1 sequence of 2000 keys     9.9  12.1  16.5        1 of 30000 keys     19.7  16.8  18.8
//   16 of 2000                 14.1  15.7  18.3        32 of 8000 to 500   49.9  47.0  44.5
//   1 of 8000                  10.4  12.2  16.4        16 of 32000          120   111   107
// With 256 dims a workgroup's own time counts for more (1 and 32 sequences, one chunk and chunks of 256: 300 keys 10.7, 11.0 and 12.7, 14.1;
// 500 keys 13.3, 13.3 and 13.0, 14.3; 1000 keys 18.5, 18.7 and 13.0, 17.8): one chunk up to 512 keys, chunks of
// 256 up to 4096 (1, 4, 16, 48 sequences of 3000 keys and fewer 13.2, 13.4, 24.9, 36.1, with chunks of 512 16.7, 16.9, 22.7, 38.0; with 128
// dims 10.0, 11.7, 20.4, 33.9 and 12.2, 12.5, 17.7, 36.1, and drafted rows, which have more to join, lose more).
// It goes by max_len, not by the lengths, which the host does not know, nor by the window.  So a capacity far above the lengths costs: one
// sequence of 128 dims with max_len 131072 and its own length, 700 keys 14.4 and 9.3, 2000 keys 16.8 and 9.9, 8192 keys 17.7 and 12.2.  And a
// window has the chunks of max_len and their join: of 8192 keys a window of 128, with max_len 8192 and 131072, 8.6 and 8.9 (128 keys in one chunk 5.6),
// of 1024 12.0 and 16.6; 32 such sequences 9.8 and 9.8 (5.8), 15.8 and 18.5.
int chunk_of(int max_len, int dim) {
    const int one = dim == 256 ? 512 : 1024;
    if (max_len <= one) return one;
    int c = max_len <= (dim == 256 ? 4096 : 2048) ? 256 : 512;
    while ((int64_t)c * kChunks < max_len) c *= 2;
    return c;
}
int chunks_of(int max_len, int dim) { return (max_len + chunk_of(max_len, dim) - 1) / chunk_of(max_len, dim); }

// units of work at most, and the workgroups that are resident at once
uint64_t units_of(const AttnArgs& a, int nt) { return (uint64_t)a.s.n * a.kv.heads * ((a.max_rows * a.share + 16 * nt - 1) / (16 * nt)) * a.chunks; }
uint64_t resident(int D, int NT, bool wide, int nw) { return (uint64_t)device_cu_count() * (occupancy(D, NT, wide) * 4 / nw); }

template <int D, int NT, bool WIDE, int NW>
int launch(AttnArgs& a, hipStream_t s) {
    a.groups = (a.max_rows * a.share + 16 * NT - 1) / (16 * NT);
    const uint64_t most = units_of(a, NT), joins = (uint64_t)a.rows * a.heads * (D / 64);
    if (most > 0x7fffffff) return QMM_ERR_SHAPE;
    const uint64_t grid = std::min(most, resident(D, NT, WIDE, NW));
    if (!grid_fits(grid, 64 * NW) || !grid_fits(joins, 64)) return QMM_ERR_SHAPE;
    hipLaunchKernelGGL((k_attn_kv<D, NT, WIDE, NW>), dim3((unsigned)grid), dim3(64 * NW), 0, s, a);
    QMM_LAUNCH_CHECK();
    if (a.chunks > 1) {
        hipLaunchKernelGGL((k_attn_join<D>), dim3((unsigned)joins), dim3(64), 0, s, a);
        QMM_LAUNCH_CHECK();
    }
    return QMM_OK;
}

// Waves of a workgroup: four; eight where the keys are one chunk (few workgroups, whose own time counts) and registers leave room for two
// waves a SIMD (700 keys of one sequence, 128 dims: 9.2 µs, with four 11.1).  A row's bits follow from it, so this must not go by NT, which goes by the rows of a call.
constexpr bool eight(int D, bool wide) { return D < 256 || !wide; }
template <int D, int NT, bool WIDE>
int launch(AttnArgs& a, hipStream_t s) {
    if constexpr (eight(D, WIDE)) {
        static_assert(occupancy(D, NT, WIDE) >= 2, "");
        if (a.chunks == 1) return launch<D, NT, WIDE, 8>(a, s);
    }
    return launch<D, NT, WIDE, 4>(a, s);
}

// Rows of a group: 16, 32, 48 or 64, what covers a sequence's, so that the cache is read and converted once; fewer where operands and sums
// would not fit 256 registers, and 16 where the units that this makes are all resident at once (then a workgroup's own time counts).  In
// µs, groups of 16 rows and of more:
//   dim 64, 40 rows a kv head, 8 kv heads: 1 sequence of 700 keys  8.2  12.7,  16 of 700  10.4  13.0,  1 of 8000  12.6  14.1,
//                                          4 of 8000  25.4  19.3,  1 of 30000  25.0  20.1,  16 of 8000 to 500  47.8  40.4
//   dim 128, 32 rows, 4 kv heads:          1 of 8000  12.9  15.3,  4 of 8000  17.1  17.4,  32 of 32000 to 2000  185  146
template <int D>
int launch_rows(AttnArgs& a, bool wide, hipStream_t s) {
    int f = a.max_rows * a.share;
    if (units_of(a, 1) <= resident(D, 1, wide, a.chunks == 1 && eight(D, wide) ? 8 : 4)) f = 16;
    if (f <= 16 || D == 256 || (wide && D == 128)) return wide ? launch<D, 1, true>(a, s) : launch<D, 1, false>(a, s);
    if constexpr (D == 64)
        if (wide && (f > 32 && f <= 48)) return launch<D, 3, true>(a, s);
    if (f <= 32 || wide || D == 128) {
        if constexpr (D == 128) return launch<D, 2, false>(a, s);
        if constexpr (D == 64) return wide ? launch<D, 2, true>(a, s) : launch<D, 2, false>(a, s);
    }
    if constexpr (D == 64) return f <= 48 || (f > 64 && f <= 96) ? launch<D, 3, false>(a, s) : launch<D, 4, false>(a, s);
    return QMM_ERR_SHAPE;                                // not reached
}

}  // namespace
}  // namespace qmm

using namespace qmm;

extern "C" {

size_t qmm_attn_kv_ws_bytes(int rows, int heads, int dim, int max_len) {
    if (rows <= 0 || heads <= 0 || max_len <= 0 || max_len > kMaxLen || (dim != 64 && dim != 128 && dim != 256)) return 0;
    const int n = chunks_of(max_len, dim);
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
    a.chunk = chunk_of(max_len, kv->dim);
    a.chunks = chunks_of(max_len, kv->dim);
    for (a.lgc = 0; 1 << a.lgc != a.chunk;) ++a.lgc;
    a.part = (float*)ws;
    a.ml = a.part + (need ? (size_t)rows * heads * a.chunks * kv->dim : 0);
    a.q_bf = qb; a.out_bf = ob;
    a.out_vec = aligned(out, ob ? 8 : 16) && ldo % 4 == 0;
    hipStream_t s = (hipStream_t)stream;
    const bool wide = !qb || !ob;
    switch (kv->dim) {
        case 64: return launch_rows<64>(a, wide, s);
        case 128: return launch_rows<128>(a, wide, s);
        default: return launch_rows<256>(a, wide, s);
    }
}

}  // extern "C"
