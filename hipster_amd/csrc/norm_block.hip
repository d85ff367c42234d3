// norm_block.hip -- what stands between two blocks of a layer, in one pass over the row (beside the plain
// residual add + norm of act.hip):
//
//   p = y / rms(y) * wy          the norm after the block (wy NULL: p = y)
//   p = p * act(gate)            the block's gate, one per token, per channel or per value (none: 1)
//   xo = x + alpha p             the residual, scaled
//   xn = xo / rms(xo) * w        the next block's norm: bf16, f32 with its q8, or MXFP4 rows
//
// rms(v) = sqrt(sum(v^2) / n + eps).  A row is held in registers between its two sums, so x, y and the gate are
// read once and xo and xn written once; HBM bounds it (one row: the two reductions' latency).  A thread
// holds C pieces of V values, 4 (n % 4 == 0) or 1; every load is issued before the first sum.  Sums are f32 in a fixed
// order: per thread, by halves of the wave, wave by wave.  Threads and V go by n alone, so a row's bits depend on
// nothing but the row, whatever the alignment of its arrays and their strides.
//
// 2048 x 5120 with a bf16 gate per value: 37 us (28 for its 147 MB at a large copy's rate), 30 from caches, 45 with f32 and q8
// out; one row 6.6, one after another (4.3 with one gate).  Rows that start anywhere and lie an odd number of values apart: the same.
//
// Threads go by the row's length alone, since they set the order of its sums; pieces are as few as cover it (2048 rows, us):
//   256 threads up to five pieces: 5120 values 37.5 (512 threads with three: 41.3); with a sixth a wave has more
//     than 128 registers, three a SIMD instead of four: 5248 values 49.4, 512 threads with three 41.8
//   512 threads up to 8192 values: 55.5 (1024 with two: 68)
//   1024 beyond: 8320 values 82 (512 with five would take 65, in another order of sums)
// One row alone would like more threads (5120 values: 640 with two 4.8 against 6.6), 300 rows too (9.3 against 10.7).
#include "mx.hpp"

namespace qmm {
namespace {

constexpr int kNbMaxN = 16384;

enum NbOut { kNbBf16, kNbQ8, kNbMx };

struct NbArgs {
    const float* x; const void* y; const float* wy; const float* w; float* xo;
    const void* gate;
    size_t ldy, ldg;
    uint16_t* xb; float* xn; qmm_xq8 q8; qmm_xmx mx;
    int n, y_bf, gate_bf, act, per_value;
    float alpha, eps;
};

// four values in memory, at the alignment of one: a vector access may have any (the compiler emits the same
// instructions as for aligned ones)
typedef uint32_t nb_u4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t nb_u2 __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t nb_u1 __attribute__((aligned(1)));
typedef uint16_t nb_h1 __attribute__((aligned(1)));

// V values at p + i (16-byte or 8-byte access, or one value); past the row: the address clamped, the value unused
template <int V>
__device__ __forceinline__ void nb_load(float (&v)[V], const void* p, int i, int n, bool bf) {
    if constexpr (V == 4) {
        const int k = min(i, n - 4);
        if (bf) {
            const nb_u2 r = *(const nb_u2*)((const uint16_t*)p + k);
            v[0] = __uint_as_float(r.x << 16); v[1] = __uint_as_float(r.x & 0xffff0000u);
            v[2] = __uint_as_float(r.y << 16); v[3] = __uint_as_float(r.y & 0xffff0000u);
        } else {
            const nb_u4 r = *(const nb_u4*)((const float*)p + k);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(r[j]);
        }
    } else {
        const int k = min(i, n - 1);
        v[0] = bf ? bf2f(((const uint16_t*)p)[k]) : ((const float*)p)[k];
    }
}

__device__ __forceinline__ void nb_store(float* p, const float (&v)[4]) {
    *(nb_u4*)p = nb_u4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
}

__device__ __forceinline__ float nb_act(float z, int act) {
    if (act == 0) return z;
    const float s = 1.f / (1.f + expf(-z));
    return act == 1 ? s : z * s;
}

// the workgroup's sum, in every thread: half-waves by the xor tree, then their sums in order
template <int NT>
__device__ __forceinline__ float nb_sum(float v, float* part) {
    v = hw32_sum(v);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = part[0];
#pragma unroll
    for (int i = 1; i < NT / 32; ++i) s += part[i];
    return s;
}

template <int NT, int V, int C, NbOut OUT>
__global__ void __launch_bounds__(NT) k_norm_block(NbArgs a) {
    __shared__ float part[2][NT / 32];
    const size_t t = blockIdx.x;
    const int n = a.n, tid = threadIdx.x;
    const float* x = a.x + t * n;
    const void* y = a.y_bf ? (const void*)((const uint16_t*)a.y + t * a.ldy) : (const void*)((const float*)a.y + t * a.ldy);
    const void* gr = a.gate_bf ? (const void*)((const uint16_t*)a.gate + t * a.ldg) : (const void*)((const float*)a.gate + t * a.ldg);
    float xv[C][V], yv[C][V], wy[C][V], gv[C][V], wv[C][V];
    float g1[1] = {1.f};
    if (a.gate && !a.per_value) nb_load<1>(g1, gr, 0, 1, a.gate_bf);
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int i = V * (tid + NT * c);
        nb_load<V>(yv[c], y, i, n, a.y_bf);
        nb_load<V>(xv[c], x, i, n, false);
        if (a.wy) nb_load<V>(wy[c], a.wy, i, n, false);
        if (a.gate && a.per_value) nb_load<V>(gv[c], gr, i, n, a.gate_bf);
        nb_load<V>(wv[c], a.w, i, n, false);
    }
    if (a.wy) {
        float ss = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int k = 0; k < V; ++k) ss = V * (tid + NT * c) + k < n ? fmaf(yv[c][k], yv[c][k], ss) : ss;
        const float rs = 1.f / sqrtf(nb_sum<NT>(ss, part[0]) / (float)n + a.eps);
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int k = 0; k < V; ++k) yv[c][k] = yv[c][k] * rs * wy[c][k];
    }
    float ss = 0.f;
    const float g = a.gate && !a.per_value ? nb_act(g1[0], a.act) : 1.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int i = V * (tid + NT * c);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            float p = yv[c][k];
            if (a.gate) p *= a.per_value ? nb_act(gv[c][k], a.act) : g;
            xv[c][k] = i + k < n ? fmaf(a.alpha, p, xv[c][k]) : 0.f;
            ss = fmaf(xv[c][k], xv[c][k], ss);
        }
        if (i < n) {
            if constexpr (V == 4) nb_store(a.xo + t * n + i, xv[c]);
            else a.xo[t * n + i] = xv[c][0];
        }
    }
    const float rs = 1.f / sqrtf(nb_sum<NT>(ss, part[1]) / (float)n + a.eps);
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int i = V * (tid + NT * c);
        float o[V];
#pragma unroll
        for (int k = 0; k < V; ++k) o[k] = i + k < n ? xv[c][k] * rs * wv[c][k] : 0.f;
        if constexpr (OUT == kNbBf16) {
            if (i < n) {
                if constexpr (V == 4)
                    *(nb_u2*)(a.xb + t * n + i) = nb_u2{mx_bf16x2(o[0], o[1]), mx_bf16x2(o[2], o[3])};
                else a.xb[t * n + i] = (uint16_t)mx_bf16x2(o[0], 0.f);
            }
        } else if constexpr (OUT == kNbQ8) {             // n % 32 == 0: a block's lanes are in the row together
            float am = fabsf(o[0]);
#pragma unroll
            for (int k = 1; k < V; ++k) am = fmaxf(am, fabsf(o[k]));
            am = V == 4 ? g8_max(am) : g32_max(am);
            const float d = am / 127.f, id = am > 0.f ? 127.f / am : 0.f;
            int q[V], sum = 0;
#pragma unroll
            for (int k = 0; k < V; ++k) { q[k] = __float2int_rn(o[k] * id); sum += q[k]; }
            sum = V == 4 ? g8_isum(sum) : g32_isum(sum);
            if (i < n) {
                if constexpr (V == 4) {
                    nb_store(a.xn + t * n + i, o);
                    *(nb_u1*)(a.q8.q + t * n + i) = (uint32_t)(q[0] & 0xff) | ((uint32_t)(q[1] & 0xff) << 8) | ((uint32_t)(q[2] & 0xff) << 16) |
                                                       ((uint32_t)q[3] << 24);
                } else {
                    a.xn[t * n + i] = o[0];
                    a.q8.q[t * n + i] = (int8_t)q[0];
                }
                if ((i & 31) == 0) {
                    const size_t sb = (t * n + i) >> 5;
                    const float s = d * (float)sum;
                    a.q8.d[sb] = d; a.q8.s[sb] = s;
                    if (a.q8.ds) ((float2*)a.q8.ds)[sb] = make_float2(d, s);
                }
            }
        } else {                                         // past the row: code 0; whole blocks there: scale byte 0
            const int K128 = mx_steps(n);
            int m = 0;
#pragma unroll
            for (int k = 0; k < V; ++k) m = max(m, __float_as_int(o[k]) & 0x7fffffff);
            if constexpr (V == 4) {
                m = max(m, dpp_i<kDppXor1>(m)); m = max(m, dpp_i<kDppXor2>(m)); m = max(m, dpp_i<kDppHalfMirror>(m));
            } else {
#pragma unroll
                for (int s = 16; s > 0; s >>= 1) m = max(m, __shfl_xor(m, s, 64));
            }
            const int byte = mx_scale_byte(m);
            const float inv = mx_inverse(byte);
            if (i < K128 * 128) {                        // uniform over a block's lanes
                uint8_t* q = a.mx.q + t * K128 * 64 + (i >> 1);
                if constexpr (V == 4) {
                    uint32_t b = 0;
                    if (byte != 255) b = mx_codes2<1>(mx_codes2<0>(0u, o[0] * inv, o[1] * inv), o[2] * inv, o[3] * inv);
                    *(nb_h1*)q = (uint16_t)b;
                } else {
                    const float u = o[0] * inv, u1 = __int_as_float(dpp_i<kDppXor1>(__float_as_int(u)));
                    if ((i & 1) == 0) *q = (uint8_t)(byte == 255 ? 0u : mx_codes2<0>(0u, u, u1));
                }
                if ((i & 31) == 0) a.mx.e[t * K128 * 4 + (i >> 5)] = (uint8_t)byte;
            }
        }
    }
}

bool misaligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }

// the checks that every output form shares, and the arguments laid out
int nb_args(const float* x, const void* y, int y_dtype, size_t ldy, const float* wy, const qmm_gate* gate, float alpha, float* xo, const float* w,
            int T, int n, float eps, NbArgs& a) {
    if (!w || (T != 0 && (!x || !y || !xo))) return QMM_ERR_NULL;
    if (y_dtype != QMM_F32 && y_dtype != QMM_BF16) return QMM_ERR_FORMAT;
    if (T < 0 || n < 1 || n > kNbMaxN || ldy < (size_t)n) return QMM_ERR_SHAPE;
    a = NbArgs{};
    if (gate && gate->g) {
        if (gate->dtype != QMM_F32 && gate->dtype != QMM_BF16) return QMM_ERR_FORMAT;
        if (gate->act < 0 || gate->act > 2) return QMM_ERR_ARG;
        if (gate->per_value && gate->ld != 0 && gate->ld < (size_t)n) return QMM_ERR_SHAPE;
        if (misaligned(gate->g, gate->dtype == QMM_BF16 ? 2 : 4)) return QMM_ERR_ARG;
        a.gate = gate->g; a.gate_bf = gate->dtype == QMM_BF16; a.act = gate->act; a.per_value = gate->per_value != 0; a.ldg = gate->ld;
    }
    if (misaligned(x, 4) || misaligned(xo, 4) || misaligned(wy, 4) || misaligned(w, 4) || misaligned(y, y_dtype == QMM_BF16 ? 2 : 4)) return QMM_ERR_ARG;
    a.x = x; a.y = y; a.wy = wy; a.w = w; a.xo = xo; a.ldy = ldy; a.n = n; a.y_bf = y_dtype == QMM_BF16; a.alpha = alpha; a.eps = eps;
    return QMM_OK;
}

template <NbOut OUT>
int nb_launch(const NbArgs& a, int T, hipStream_t s) {
    if (T == 0) return QMM_OK;
    const int len = OUT == kNbMx ? mx_steps(a.n) * 128 : a.n;      // values written per row
    const dim3 grid((unsigned)T);
#define QMM_NB(NT, V, C) do { \
        if (!grid_fits((uint64_t)T, NT)) return QMM_ERR_SHAPE; \
        hipLaunchKernelGGL((k_norm_block<NT, V, C, OUT>), grid, dim3(NT), 0, s, a); \
    } while (0)
    const auto pieces = [&](int threads) { return (len + 4 * threads - 1) / (4 * threads); };
    if (a.n % 4 != 0) {
        if (len <= 4096) QMM_NB(1024, 1, 4);
        else QMM_NB(1024, 1, 16);
    } else if (len <= 5120) {
        switch (pieces(256)) {
            case 1: QMM_NB(256, 4, 1); break;
            case 2: QMM_NB(256, 4, 2); break;
            case 3: QMM_NB(256, 4, 3); break;
            case 4: QMM_NB(256, 4, 4); break;
            default: QMM_NB(256, 4, 5);
        }
    } else if (len <= 8192) {
        if (pieces(512) <= 3) QMM_NB(512, 4, 3);
        else QMM_NB(512, 4, 4);
    } else {
        if (pieces(1024) <= 3) QMM_NB(1024, 4, 3);
        else QMM_NB(1024, 4, 4);
    }
#undef QMM_NB
    QMM_LAUNCH_CHECK();
    return QMM_OK;
}

}  // namespace
}  // namespace qmm

using namespace qmm;

extern "C" {

int qmm_postnorm_add_rmsnorm_bf16(const float* x, const void* y, int y_dtype, size_t ldy, const float* wy, const qmm_gate* gate, float alpha,
                                  float* xo, const float* w, uint16_t* xb, int T, int n, float eps, void* stream) {
    NbArgs a;
    const int st = nb_args(x, y, y_dtype, ldy, wy, gate, alpha, xo, w, T, n, eps, a);
    if (st != QMM_OK) return st;
    if (T != 0 && !xb) return QMM_ERR_NULL;
    if (misaligned(xb, 2)) return QMM_ERR_ARG;
    a.xb = xb;
    return nb_launch<kNbBf16>(a, T, (hipStream_t)stream);
}

int qmm_postnorm_add_rmsnorm_quant(const float* x, const void* y, int y_dtype, size_t ldy, const float* wy, const qmm_gate* gate, float alpha,
                                   float* xo, const float* w, float* xn, qmm_xq8 xq, int T, int n, float eps, void* stream) {
    NbArgs a;
    const int st = nb_args(x, y, y_dtype, ldy, wy, gate, alpha, xo, w, T, n, eps, a);
    if (st != QMM_OK) return st;
    if (T != 0 && (!xn || !xq.q || !xq.d || !xq.s)) return QMM_ERR_NULL;
    if (n % 32 != 0) return QMM_ERR_SHAPE;
    if (misaligned(xn, 4) || misaligned(xq.d, 4) || misaligned(xq.s, 4) || misaligned(xq.ds, 8)) return QMM_ERR_ARG;
    a.xn = xn; a.q8 = xq;
    return nb_launch<kNbQ8>(a, T, (hipStream_t)stream);
}

int qmm_postnorm_add_rmsnorm_mxfp4(const float* x, const void* y, int y_dtype, size_t ldy, const float* wy, const qmm_gate* gate, float alpha,
                                   float* xo, const float* w, qmm_xmx xq, int T, int n, float eps, void* stream) {
    NbArgs a;
    const int st = nb_args(x, y, y_dtype, ldy, wy, gate, alpha, xo, w, T, n, eps, a);
    if (st != QMM_OK) return st;
    if (T != 0 && (!xq.q || !xq.e)) return QMM_ERR_NULL;
    a.mx = xq;
    return nb_launch<kNbMx>(a, T, (hipStream_t)stream);
}

}  // extern "C"
