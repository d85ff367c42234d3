// mx.hpp -- the MXFP4 format on gfx950: layouts and device helpers shared by mx_quant.hip and mx_gemm.hip.
//
// A row of K values is blocks of 32: codes e2m1 (sign, 2 exponent bits, 1 mantissa bit: 0, 0.5, 1, 1.5, 2, 3,
// 4, 6) and one scale byte E8M0, 2^(byte - 127), 255 = NaN.  Rows are padded to K128 = ceil(K / 128) steps of
// 128 values, the padding being code 0 with scale byte 0, so no kernel masks K.
//
//   rows (activations, and weights before packing), qmm_xmx:
//     q [R][K128][64 bytes]  value 2i of the step in the low half of byte i, value 2i + 1 in the high half
//     e [R][K128][4 bytes]   one scale byte per block
//   packed weights (qmm_pack_mxfp4): per 16 rows one tile strip, strips in row order
//     codes  [K128][64 lanes][16 bytes]         lane l: row l % 16, block l / 16 of the step
//     scales [ceil(K128 / 4)][64 lanes][4 bytes] the four bytes: the lane's block of four successive steps
//
// The strip is in the order of the scaled matrix instructions: a lane supplies 32 codes of one row, a block, and the
// block's scale in one byte of a register (which byte, the instruction says).  So a wave reads half a step of two
// strips as two runs of 512 bytes and four steps' scales as one dword per lane, with no shuffle.
//
// The instruction's sum of products is exact to f32 rounding for fp4 operands (measured: within 1.3 * 2^-24 of the sum of
// magnitudes with block scales spread over 2^+-40); for fp8 operands it is not (products 2^15 below a group's largest
// are dropped), which is why activations are fp4 too.
#pragma once
#include "qmm_common.hpp"

namespace qmm {

typedef int mx_v8i __attribute__((ext_vector_type(8)));
typedef float mx_v4f __attribute__((ext_vector_type(4)));
typedef float mx_v16f __attribute__((ext_vector_type(16)));

constexpr int kMxMaxK = 1 << 24;                 // a strip's byte offsets stay in 32 bits
constexpr int kMxMaxRows = 0x7fffff00;                // of a weight or a GEMM: a tile past the last row stays an int
constexpr int kMxFp4 = 4;                        // the instruction's number for e2m1

__host__ __device__ __forceinline__ int mx_steps(int K) { return (K + 127) >> 7; }
__host__ __device__ __forceinline__ int mx_groups(int K128) { return (K128 + 3) >> 2; }
__host__ __device__ __forceinline__ uint32_t mx_strip_bytes(int K128) { return (uint32_t)K128 * 1024u + (uint32_t)mx_groups(K128) * 256u; }

// the scale byte of a block whose largest |x| has the bits m (as an integer: NaN above infinity above all):
// the exponent field less two, clamped at 0; 255 where m is not finite
__device__ __forceinline__ int mx_scale_byte(int m) { return m < 0x7f800000 ? max((m >> 23) - 2, 0) : 255; }
// what its values are multiplied with before their rounding: 2^(127 - byte); 0 for byte 255 (codes 0)
__device__ __forceinline__ float mx_inverse(int byte) { return __int_as_float(byte == 255 ? 0 : (254 - byte) << 23); }
// codes of two scaled values into byte B of old
template <int B>
__device__ __forceinline__ uint32_t mx_codes2(uint32_t old, float lo, float hi) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(old, lo, hi, 1.f, B);
}

// acc += W . A^T over half a step (64 values), 32 x 32: w and a the two operands' 16 bytes (lane l: row l % 32, block
// l / 32 of the half), their scales in byte BW of sw and byte BA of sa.  acc[e] of lane l: weight row
// 8 (e / 4) + 4 (l / 32) + e % 4, activation row l % 32.
template <int BW, int BA>
__device__ __forceinline__ mx_v16f mx_mfma32(const uint4& w, const uint4& a, mx_v16f acc, uint32_t sw, uint32_t sa) {
    const mx_v8i vw = {(int)w.x, (int)w.y, (int)w.z, (int)w.w, 0, 0, 0, 0};
    const mx_v8i va = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(vw, va, acc, kMxFp4, kMxFp4, BW, (int)sw, BA, (int)sa);
}

// two values rounded to bf16 (to nearest even; NaN stays NaN), the first in the low half
__device__ __forceinline__ uint32_t mx_bf16x2(float lo, float hi) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)lo, (__bf16)hi});
}

// four outputs of one activation row: weight rows n .. n + 3 of D[m][N]
template <bool BF>
__device__ __forceinline__ void mx_store4(void* D, size_t at, const mx_v4f& v, int left, bool vec) {
    if constexpr (BF) {
        uint16_t* d = (uint16_t*)D + at;
        if (vec && left >= 4) {
            *(uint2*)d = make_uint2(mx_bf16x2(v[0], v[1]), mx_bf16x2(v[2], v[3]));
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i < left) d[i] = (uint16_t)mx_bf16x2(v[i], 0.f);
        }
    } else {
        float* d = (float*)D + at;
        if (vec && left >= 4) {
            *(mx_v4f*)d = v;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i < left) d[i] = v[i];
        }
    }
}

}  // namespace qmm
