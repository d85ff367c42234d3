// kv_cache.hip -- rows of keys and values into the pages of an MXFP4 cache, and back (layout: qmm_kv_mxfp4 in hipster_qmm.h).
//
//   k_kv_write   rows of f32 or bf16 -> codes and scale bytes at their tokens' places
//   k_kv_read    the values at the rows' places -> rows of f32 or bf16
//
// A token of one head is a row of MXFP4 as quantize_mxfp4 makes it, dim / 2 bytes of codes and dim / 32 of scales, keys and values
// alike: writing a token touches no byte of another one, and a wave that reads 16 tokens of a head reads one run of memory.
//
// Both move each byte once.  A lane has 8 values (a quarter of a block, 16 bytes of bf16); a wave has 64 or 256 such pieces of one row, the
// keys' pieces first, then the values', so that its row, sequence and page are found once, in registers of the whole wave.  4700 rows of 8 heads
// of 128 in bf16, 24.6 MB each: written in 8.9 us, read in 7.6 (2.8 and 3.2 TB/s): a launch, and a chain of three loads (offsets, page, data).
#include "attn.hpp"

namespace qmm {
namespace {

constexpr int kWaves = 4;

struct KvArgs {
    qmm_kv_mxfp4 kv;
    qmm_seqs s;
    int lg, rows, parts;                                 // parts: waves per row
    size_t ldk, ldv;
};

// Row, page (-1: outside the cache) and place in it of a wave's row; false: the row has no place
__device__ __forceinline__ bool place(const KvArgs& a, int row, int& page, int& at) {
    SeqSpan q;
    const int b = seq_of_row(a.s.cu, a.s.lens, a.s.n, a.rows, row, q);
    if (b < 0) return false;
    const int pos = q.len - q.m + (row - q.r0);
    if (pos < 0 || (pos >> a.lg) >= a.s.ld) return false;
    page = a.s.table[(size_t)b * a.s.ld + (pos >> a.lg)];
    if ((unsigned)page >= (unsigned)a.kv.pages) page = -1;
    at = pos & (a.kv.page - 1);
    return true;
}

// eight values at p as they lie in memory (bf16: two a word) and as f32
template <bool BF>
struct Eight { uint32_t w[BF ? 4 : 8]; };
template <bool BF, bool VEC>
__device__ __forceinline__ void get(const void* src, size_t from, Eight<BF>& v) {
    if constexpr (BF && VEC) {
        const uint4 r = *(const uint4*)((const uint16_t*)src + from);
        v.w[0] = r.x; v.w[1] = r.y; v.w[2] = r.z; v.w[3] = r.w;
    } else if constexpr (BF) {
        const uint16_t* p = (const uint16_t*)src + from;
#pragma unroll
        for (int i = 0; i < 4; ++i) v.w[i] = p[2 * i] | ((uint32_t)p[2 * i + 1] << 16);
    } else if constexpr (VEC) {
        const uint4 r = *(const uint4*)((const float*)src + from), s = *(const uint4*)((const float*)src + from + 4);
        v.w[0] = r.x; v.w[1] = r.y; v.w[2] = r.z; v.w[3] = r.w; v.w[4] = s.x; v.w[5] = s.y; v.w[6] = s.z; v.w[7] = s.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v.w[i] = ((const uint32_t*)src)[from + i];
    }
}
template <bool BF>
__device__ __forceinline__ float f32_of(const Eight<BF>& v, int i) {
    if constexpr (BF) return __uint_as_float((i & 1) ? v.w[i / 2] & 0xffff0000u : v.w[i / 2] << 16);
    else return __uint_as_float(v.w[i]);
}

template <bool BF, bool VEC, int PP>
__global__ void __launch_bounds__(64 * kWaves) k_kv_write(const void* __restrict__ k, const void* __restrict__ v, KvArgs a) {
    const uint32_t item = __builtin_amdgcn_readfirstlane(blockIdx.x * kWaves + (threadIdx.x >> 6));
    const uint32_t row = item / (uint32_t)a.parts;
    if (row >= (uint32_t)a.rows) return;
    const int D = a.kv.dim, C = a.kv.heads * D / 8;      // pieces of the row's keys
    const int c0 = (int)(item - row * a.parts) * (64 * PP) + (threadIdx.x & 63);
    Eight<BF> x[PP];
#pragma unroll
    for (int i = 0; i < PP; ++i) {                       // whole blocks lie past the end together
        const int c = c0 + 64 * i;
        if (c < 2 * C) get<BF, VEC>(c >= C ? v : k, (size_t)row * (c >= C ? a.ldv : a.ldk) + (size_t)(c >= C ? c - C : c) * 8, x[i]);
    }
    int page, at;
    if (!place(a, (int)row, page, at) || page < 0) return;
#pragma unroll
    for (int i = 0; i < PP; ++i) {
        const int cc = c0 + 64 * i;
        if (cc >= 2 * C) break;
        const bool val = cc >= C;
        const int c = val ? cc - C : cc;
        int m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, __float_as_int(f32_of<BF>(x[i], j)) & 0x7fffffff);
        m = max(m, dpp_i<kDppXor1>(m));                  // the block's four lanes
        m = max(m, dpp_i<kDppXor2>(m));
        const int byte = mx_scale_byte(m);
        const float inv = mx_inverse(byte);
        uint32_t code = 0;
        if (byte != 255) {                               // a NaN times 0 would not be code 0
            code = mx_codes2<0>(code, f32_of<BF>(x[i], 0) * inv, f32_of<BF>(x[i], 1) * inv);
            code = mx_codes2<1>(code, f32_of<BF>(x[i], 2) * inv, f32_of<BF>(x[i], 3) * inv);
            code = mx_codes2<2>(code, f32_of<BF>(x[i], 4) * inv, f32_of<BF>(x[i], 5) * inv);
            code = mx_codes2<3>(code, f32_of<BF>(x[i], 6) * inv, f32_of<BF>(x[i], 7) * inv);
        }
        const int h = c / (D / 8), d8 = c & (D / 8 - 1);
        const size_t to = ((size_t)page * a.kv.heads + h) * a.kv.page + at;  // token of a head
        *(uint32_t*)((val ? a.kv.vq : a.kv.kq) + to * (D / 2) + d8 * 4) = code;
        if ((d8 & 3) == 0) (val ? a.kv.ve : a.kv.ke)[to * (D / 32) + d8 / 4] = (uint8_t)byte;
    }
}

template <bool BF, bool VEC, int PP>
__global__ void __launch_bounds__(64 * kWaves) k_kv_read(void* __restrict__ k, void* __restrict__ v, KvArgs a) {
    const uint32_t item = __builtin_amdgcn_readfirstlane(blockIdx.x * kWaves + (threadIdx.x >> 6));
    const uint32_t row = item / (uint32_t)a.parts;
    if (row >= (uint32_t)a.rows) return;
    int page, at;
    if (!place(a, (int)row, page, at)) return;
    const int D = a.kv.dim, C = a.kv.heads * D / 8;
    const int c0 = (int)(item - row * a.parts) * (64 * PP) + (threadIdx.x & 63);
    uint32_t code[PP], byte[PP];
#pragma unroll
    for (int i = 0; i < PP; ++i) {
        const int cc = c0 + 64 * i;
        if (cc >= 2 * C) break;
        const bool val = cc >= C;
        const int c = val ? cc - C : cc, h = c / (D / 8), d8 = c & (D / 8 - 1);
        const size_t from = ((size_t)max(page, 0) * a.kv.heads + h) * a.kv.page + at;
        code[i] = *(const uint32_t*)((val ? a.kv.vq : a.kv.kq) + from * (D / 2) + d8 * 4);
        byte[i] = (val ? a.kv.ve : a.kv.ke)[from * (D / 32) + d8 / 4];
    }
#pragma unroll
    for (int i = 0; i < PP; ++i) {
        const int cc = c0 + 64 * i;
        if (cc >= 2 * C) break;
        const bool val = cc >= C;
        const int c = val ? cc - C : cc;
        // the conversion reads the scale's exponent field: 2^(byte - 127), 255 NaN
        const float s = __uint_as_float((page < 0 || byte[i] >= kMxNan ? 255u : byte[i]) << 23);
        uint32_t w[4];                                   // two significant bits: exact in bf16
        w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code[i], s, 0));
        w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code[i], s, 1));
        w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code[i], s, 2));
        w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code[i], s, 3));
        const size_t to = (size_t)row * (val ? a.ldv : a.ldk) + (size_t)c * 8;
        if constexpr (BF) {
            uint16_t* p = (uint16_t*)(val ? v : k) + to;
            if constexpr (VEC) {
                *(uint4*)p = make_uint4(w[0], w[1], w[2], w[3]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) p[j] = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
            }
        } else {
            float* p = (float*)(val ? v : k) + to;
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = __uint_as_float((j & 1) ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
            if constexpr (VEC) {
                *(float4*)p = make_float4(x[0], x[1], x[2], x[3]);
                *(float4*)(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) p[j] = x[j];
            }
        }
    }
}

// checks that both calls share; *go: there are rows
int prepare(const void* k, size_t ldk, const void* v, size_t ldv, int dtype, const qmm_kv_mxfp4* kv, const qmm_seqs* s, int rows, KvArgs& a, bool& vec,
            bool& wide, unsigned& grid, bool& go) {
    go = false;
    if (dtype != QMM_F32 && dtype != QMM_BF16) return QMM_ERR_FORMAT;
    if (rows < 0) return QMM_ERR_SHAPE;
    if (rows == 0) return QMM_OK;
    if (!k || !v) return QMM_ERR_NULL;
    if (const int st = kv_check(kv, s, &a.lg)) return st;
    const size_t n = (size_t)kv->heads * kv->dim;
    if (ldk < n || ldv < n) return QMM_ERR_SHAPE;
    const size_t size = dtype == QMM_BF16 ? 2 : 4;
    if (!aligned(k, size) || !aligned(v, size)) return QMM_ERR_ARG;
    a.kv = *kv; a.s = *s; a.rows = rows; a.ldk = ldk; a.ldv = ldv;
    // A wave has four times 64 pieces of a row where that leaves a round of waves for every SIMD, else one (few rows: latency counts).
    // 8 heads of 128, write and read, in µs with one and four: 24 rows 4.7 and 6.3, 512 rows 6.1 and 7.3, 8192 rows 28 and 22.5
    wide = (uint64_t)rows * ((2 * n / 8 + 255) / 256) >= 4096;
    a.parts = (int)(wide ? (2 * n / 8 + 255) / 256 : (2 * n / 8 + 63) / 64);
    vec = aligned(k, 16) && aligned(v, 16) && ldk * size % 16 == 0 && ldv * size % 16 == 0;
    const uint64_t items = (uint64_t)rows * a.parts, blocks = (items + kWaves - 1) / kWaves;
    if (items > 0xffffffffu - kWaves || !grid_fits(blocks, 64 * kWaves)) return QMM_ERR_SHAPE;
    grid = (unsigned)blocks;
    go = true;
    return QMM_OK;
}

}  // namespace
}  // namespace qmm

using namespace qmm;

extern "C" {

int qmm_kv_write_mxfp4(const void* k, size_t ldk, const void* v, size_t ldv, int dtype, const qmm_kv_mxfp4* kv, const qmm_seqs* seqs, int rows,
                       void* stream) {
    KvArgs a;
    bool vec, wide, go;
    unsigned grid;
    const int st = prepare(k, ldk, v, ldv, dtype, kv, seqs, rows, a, vec, wide, grid, go);
    if (st != QMM_OK || !go) return st;
    const dim3 g(grid), t(64 * kWaves);
    hipStream_t s = (hipStream_t)stream;
    auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, g, t, 0, s, k, v, a); };
    if (dtype == QMM_BF16 && vec) wide ? launch(k_kv_write<true, true, 4>) : launch(k_kv_write<true, true, 1>);
    else if (dtype == QMM_BF16) wide ? launch(k_kv_write<true, false, 4>) : launch(k_kv_write<true, false, 1>);
    else if (vec) wide ? launch(k_kv_write<false, true, 4>) : launch(k_kv_write<false, true, 1>);
    else wide ? launch(k_kv_write<false, false, 4>) : launch(k_kv_write<false, false, 1>);
    QMM_LAUNCH_CHECK();
    return QMM_OK;
}

int qmm_kv_read_mxfp4(const qmm_kv_mxfp4* kv, const qmm_seqs* seqs, void* k, size_t ldk, void* v, size_t ldv, int dtype, int rows, void* stream) {
    KvArgs a;
    bool vec, wide, go;
    unsigned grid;
    const int st = prepare(k, ldk, v, ldv, dtype, kv, seqs, rows, a, vec, wide, grid, go);
    if (st != QMM_OK || !go) return st;
    const dim3 g(grid), t(64 * kWaves);
    hipStream_t s = (hipStream_t)stream;
    auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, g, t, 0, s, k, v, a); };
    if (dtype == QMM_BF16 && vec) wide ? launch(k_kv_read<true, true, 4>) : launch(k_kv_read<true, true, 1>);
    else if (dtype == QMM_BF16) wide ? launch(k_kv_read<true, false, 4>) : launch(k_kv_read<true, false, 1>);
    else if (vec) wide ? launch(k_kv_read<false, true, 4>) : launch(k_kv_read<false, true, 1>);
    else wide ? launch(k_kv_read<false, false, 4>) : launch(k_kv_read<false, false, 1>);
    QMM_LAUNCH_CHECK();
    return QMM_OK;
}

}  // extern "C"
