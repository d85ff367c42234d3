// mx_quant.hip -- MXFP4 rows: quantisation, the values they hold, and the packing of weights (layouts: mx.hpp).
//
//   qmm_quantize_mxfp4   rows of f32 or bf16 -> qmm_xmx
//   qmm_dequant_mxfp4    qmm_xmx -> f32 or bf16 rows
//   qmm_pack_mxfp4       qmm_xmx rows of a weight -> the strips the products read
//
// A block's scale is 2^E, E = floor(log2 amax) - 2, at least -127 (the largest binade of e2m1 starts at
// 4 = 2^2): its byte is the exponent field of amax less two, clamped at 0.  x 2^-E is exact, so a code is one
// rounding (to nearest, ties to even, saturating at 6) whatever computes it, and the codes are the
// definition's bit for bit.  amax is taken on the bits of |x| as an integer: a NaN is then the largest of all and a block
// that holds a NaN or an infinity gets the scale byte 255 (NaN), so a product shows it.
//
// All three move each byte once and are bound by HBM: a thread takes one 16-byte load of input (4 f32 or
// 8 bf16), 8 or 4 neighbouring lanes make a block and find amax by DPP.  2048 x 17408 bf16 (90 MB, 17 us at a
// large copy's rate): quantisation 23 us from memory, 16 from caches; the values back as bf16 16.
#include "mx.hpp"

namespace qmm {
namespace {

constexpr int kQThreads = 256;

// 8 lanes (f32) or 4 lanes (bf16) of a block: the largest of their integers
template <int V>
__device__ __forceinline__ int block_max(int v) {
    v = max(v, dpp_i<kDppXor1>(v));
    v = max(v, dpp_i<kDppXor2>(v));
    return V == 4 ? max(v, dpp_i<kDppHalfMirror>(v)) : v;
}

template <bool BF, bool VEC>
__global__ void __launch_bounds__(kQThreads) k_quantize_mxfp4(const void* __restrict__ x, size_t ldx, uint8_t* __restrict__ q,
                                                              uint8_t* __restrict__ e, uint32_t pieces, uint32_t per_row, int K) {
    constexpr int V = BF ? 8 : 4;                        // values per thread
    const uint32_t p = blockIdx.x * kQThreads + threadIdx.x;
    if (p >= pieces) return;                             // a row's pieces fill whole blocks: blocks leave together
    const uint32_t row = p / per_row, k = (p - row * per_row) * V;
    float v[V];
    const size_t at = (size_t)row * ldx + k;
    if (VEC && k + V <= (uint32_t)K) {
        const uint4 r = *(const uint4*)((const uint8_t*)x + at * (BF ? 2 : 4));
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (BF) {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            } else {
                v[i] = __uint_as_float(w[i]);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            v[i] = 0.f;
            if (k + i < (uint32_t)K) v[i] = BF ? bf2f(((const uint16_t*)x)[at + i]) : ((const float*)x)[at + i];
        }
    }
    int m = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) m = max(m, __float_as_int(v[i]) & 0x7fffffff);
    m = block_max<V>(m);
    const int byte = mx_scale_byte(m);
    const float inv = mx_inverse(byte);
    uint32_t c = 0;
    if (byte != 255) {                                   // a NaN times 0 would not be code 0
        c = mx_codes2<0>(c, v[0] * inv, v[1] * inv);
        c = mx_codes2<1>(c, v[2] * inv, v[3] * inv);
        if constexpr (BF) {
            c = mx_codes2<2>(c, v[4] * inv, v[5] * inv);
            c = mx_codes2<3>(c, v[6] * inv, v[7] * inv);
        }
    }
    if constexpr (BF) *(uint32_t*)(q + (size_t)p * 4) = c;
    else *(uint16_t*)(q + (size_t)p * 2) = (uint16_t)c;
    if ((p & (32 / V - 1)) == 0) e[p / (32 / V)] = (uint8_t)byte;
}

// the values of eight codes: e2m1 as the top bits of an f32 is the value times 2^-126 (codes 0 and 1 are its
// subnormals), then the block's scale; both products are exact
__device__ __forceinline__ float mx_value(uint32_t code, float scale) {
    const float v = __uint_as_float((code & 7u) << 22) * 0x1p126f * scale;
    return __uint_as_float(__float_as_uint(v) | ((code & 8u) << 28));
}

template <bool BF, bool VEC>
__global__ void __launch_bounds__(kQThreads) k_dequant_mxfp4(const uint8_t* __restrict__ q, const uint8_t* __restrict__ e, void* __restrict__ out,
                                                             uint32_t pieces, uint32_t per_row, int K, int K128) {
    const uint32_t p = blockIdx.x * kQThreads + threadIdx.x;
    if (p >= pieces) return;
    const uint32_t row = p / per_row, k = (p - row * per_row) * 8;
    const uint32_t c = *(const uint32_t*)(q + (size_t)row * K128 * 64 + k / 2);
    const uint32_t byte = e[(size_t)row * K128 * 4 + k / 32];
    const float s = byte == 0 ? 0x1p-127f : byte == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte << 23);
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = mx_value(c >> (4 * i), s);
    const size_t at = (size_t)row * K + k;
    if (VEC && k + 8 <= (uint32_t)K) {
        if constexpr (BF) {
            uint32_t w[4];                               // a value has two significant bits: its bf16 is its top half
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = (__float_as_uint(v[2 * i]) >> 16) | (__float_as_uint(v[2 * i + 1]) & 0xffff0000u);
            *(uint4*)((uint16_t*)out + at) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
            *(float4*)((float*)out + at) = make_float4(v[0], v[1], v[2], v[3]);
            *(float4*)((float*)out + at + 4) = make_float4(v[4], v[5], v[6], v[7]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (k + i < (uint32_t)K) {
                if constexpr (BF) ((uint16_t*)out)[at + i] = (uint16_t)(__float_as_uint(v[i]) >> 16);
                else ((float*)out)[at + i] = v[i];
            }
    }
}

// one wave per (strip, group of four steps): the group's four kilobytes of codes and its 256 bytes of scales
__global__ void __launch_bounds__(64) k_pack_mxfp4(const uint8_t* __restrict__ q, const uint8_t* __restrict__ e, uint8_t* __restrict__ W,
                                                   int N, int K128, uint32_t groups) {
    const uint32_t strip = blockIdx.x / groups, g = blockIdx.x - strip * groups;
    const int lane = threadIdx.x, row = (int)strip * 16 + (lane & 15), blk = lane >> 4;
    uint8_t* codes = W + (size_t)strip * mx_strip_bytes(K128);
    uint32_t sc = 0;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const int kt = 4 * (int)g + s;
        if (kt >= K128) break;                           // uniform
        uint4 c = make_uint4(0, 0, 0, 0);
        if (row < N) {
            c = *(const uint4*)(q + ((size_t)row * K128 + kt) * 64 + blk * 16);
            sc |= (uint32_t)e[((size_t)row * K128 + kt) * 4 + blk] << (8 * s);
        }
        *(uint4*)(codes + (size_t)kt * 1024 + lane * 16) = c;
    }
    *(uint32_t*)(codes + (size_t)K128 * 1024 + (size_t)g * 256 + lane * 4) = sc;
}

bool misaligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }

}  // namespace
}  // namespace qmm

using namespace qmm;

extern "C" {

size_t qmm_mxfp4_weight_bytes(int N, int K) {
    if (N <= 0 || N > kMxMaxRows || K <= 0 || K > kMxMaxK) return 0;
    return (size_t)((N + 15) / 16) * mx_strip_bytes(mx_steps(K));
}

int qmm_quantize_mxfp4(const void* x, int dtype, size_t ldx, qmm_xmx out, int rows, int K, void* stream) {
    if (rows != 0 && (!x || !out.q || !out.e)) return QMM_ERR_NULL;
    if (dtype != QMM_F32 && dtype != QMM_BF16) return QMM_ERR_FORMAT;
    if (rows < 0 || K <= 0 || K > kMxMaxK || ldx < (size_t)K) return QMM_ERR_SHAPE;
    if (misaligned(out.q, 16) || misaligned(out.e, 4) || misaligned(x, dtype == QMM_BF16 ? 2 : 4)) return QMM_ERR_ARG;
    if (rows == 0) return QMM_OK;
    const bool bf = dtype == QMM_BF16;
    const uint32_t per_row = (uint32_t)mx_steps(K) * (bf ? 16u : 32u);
    const uint64_t pieces = (uint64_t)rows * per_row;
    if (pieces > 0xffffff00u) return QMM_ERR_SHAPE;
    const bool vec = !misaligned(x, 16) && ldx % (bf ? 8 : 4) == 0;
    const dim3 grid((unsigned)((pieces + kQThreads - 1) / kQThreads)), block(kQThreads);
    hipStream_t s = (hipStream_t)stream;
    const uint32_t np = (uint32_t)pieces;
    if (bf && vec) hipLaunchKernelGGL((k_quantize_mxfp4<true, true>), grid, block, 0, s, x, ldx, out.q, out.e, np, per_row, K);
    else if (bf) hipLaunchKernelGGL((k_quantize_mxfp4<true, false>), grid, block, 0, s, x, ldx, out.q, out.e, np, per_row, K);
    else if (vec) hipLaunchKernelGGL((k_quantize_mxfp4<false, true>), grid, block, 0, s, x, ldx, out.q, out.e, np, per_row, K);
    else hipLaunchKernelGGL((k_quantize_mxfp4<false, false>), grid, block, 0, s, x, ldx, out.q, out.e, np, per_row, K);
    QMM_LAUNCH_CHECK();
    return QMM_OK;
}

int qmm_dequant_mxfp4(qmm_xmx x, void* out, int dtype, int rows, int K, void* stream) {
    if (rows != 0 && (!x.q || !x.e || !out)) return QMM_ERR_NULL;
    if (dtype != QMM_F32 && dtype != QMM_BF16) return QMM_ERR_FORMAT;
    if (rows < 0 || K <= 0 || K > kMxMaxK) return QMM_ERR_SHAPE;
    if (misaligned(x.q, 4) || misaligned(out, dtype == QMM_BF16 ? 2 : 4)) return QMM_ERR_ARG;
    if (rows == 0) return QMM_OK;
    const bool bf = dtype == QMM_BF16;
    const uint32_t per_row = (uint32_t)(K + 7) / 8;
    const uint64_t pieces = (uint64_t)rows * per_row;
    if (pieces > 0xffffff00u) return QMM_ERR_SHAPE;
    const bool vec = !misaligned(out, 16) && K % (bf ? 8 : 4) == 0;
    const dim3 grid((unsigned)((pieces + kQThreads - 1) / kQThreads)), block(kQThreads);
    hipStream_t s = (hipStream_t)stream;
    const uint32_t np = (uint32_t)pieces;
    const int K128 = mx_steps(K);
    if (bf && vec) hipLaunchKernelGGL((k_dequant_mxfp4<true, true>), grid, block, 0, s, x.q, x.e, out, np, per_row, K, K128);
    else if (bf) hipLaunchKernelGGL((k_dequant_mxfp4<true, false>), grid, block, 0, s, x.q, x.e, out, np, per_row, K, K128);
    else if (vec) hipLaunchKernelGGL((k_dequant_mxfp4<false, true>), grid, block, 0, s, x.q, x.e, out, np, per_row, K, K128);
    else hipLaunchKernelGGL((k_dequant_mxfp4<false, false>), grid, block, 0, s, x.q, x.e, out, np, per_row, K, K128);
    QMM_LAUNCH_CHECK();
    return QMM_OK;
}

int qmm_pack_mxfp4(qmm_xmx rows, void* W, int N, int K, void* stream) {
    if (!rows.q || !rows.e || !W) return QMM_ERR_NULL;
    if (N <= 0 || N > kMxMaxRows || K <= 0 || K > kMxMaxK) return QMM_ERR_SHAPE;
    if (misaligned(rows.q, 16) || misaligned(W, 16)) return QMM_ERR_ARG;
    const int K128 = mx_steps(K);
    const uint32_t groups = (uint32_t)mx_groups(K128);
    const uint64_t blocks = (uint64_t)((N + 15) / 16) * groups;
    if (!grid_fits(blocks, 64)) return QMM_ERR_SHAPE;
    hipLaunchKernelGGL(k_pack_mxfp4, dim3((unsigned)blocks), dim3(64), 0, (hipStream_t)stream, rows.q, rows.e, (uint8_t*)W, N, K128, groups);
    QMM_LAUNCH_CHECK();
    return QMM_OK;
}

}  // extern "C"
