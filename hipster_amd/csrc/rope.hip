// rope.hip -- rotary positions with several axes.
//
// Pair (a, b) of a head, pair number i of a token t:  (a c - b s, b c + a s) with the angle pos[axis(i)][t] * freq[i].
//
// The product of an int32 and an f32 has up to 55 bits: it is held as a double and the double of what that misses, taken to
// [-pi/4, pi/4] and a quadrant by pi/2 as its nearest double and the rest, and only then rounded to f32 (off by 2^-25), where sine
// and cosine are their Taylor series (rest below 2^-29).  So an angle at position 10^6 is as good as one at 1.
//
// Bound by HBM: every value is read once and written once.  A thread keeps the angles of its pairs for several heads of a token, which
// makes the 64-bit reduction (some 12 instructions a pair) small beside them; with few tokens the heads are spread over threads
// instead, as then only the chain of one thread counts.  2000 tokens of 20 heads of 256 in bf16, 41 MB: 9.4 us (4.4 TB/s; a copy of
// that size 8.0 us).
#include "attn.hpp"

namespace qmm {
namespace {

constexpr int kThreads = 256, kBatch = 4;

struct RopeArgs {
    const void* x;
    void* out;
    qmm_rope r;
    size_t ldx, ldo;
    uint32_t units, turned, groups, items;               // units of a head (the turned ones first), heads' groups of a token, threads
    int heads, per, dim;                                 // per: heads of a group
};

// cosine and sine of pos * freq
__device__ __forceinline__ void turn_of(int pos, float freq, float& c, float& s) {
    constexpr double kHalfPi = 1.57079632679489661923, kHalfPiRest = 6.12323399573676603587e-17, kTwoByPi = 0.63661977236758134308;
    const double p = (double)pos, f = (double)freq;
    const double hi = p * f, lo = fma(p, f, -hi);
    const double n = rint(hi * kTwoByPi);
    const double r = fma(-n, kHalfPiRest, fma(-n, kHalfPi, hi)) + lo;
    const int quad = (int)(n - 4.0 * floor(n * 0.25));
    const float z = (float)r, z2 = z * z;
    float sn = fmaf(z2, 2.75573192e-6f, -1.98412698e-4f);
    sn = fmaf(z2, sn, 8.33333333e-3f);
    sn = fmaf(z2, sn, -1.66666667e-1f);
    sn = fmaf(z * z2, sn, z);
    float cs = fmaf(z2, -2.75573192e-7f, 2.48015873e-5f);
    cs = fmaf(z2, cs, -1.38888889e-3f);
    cs = fmaf(z2, cs, 4.16666667e-2f);
    cs = fmaf(z2, cs, -0.5f);
    cs = fmaf(z2, cs, 1.f);
    c = (quad & 1) ? sn : cs;
    s = (quad & 1) ? cs : sn;
    if (quad == 1 || quad == 2) c = -c;
    if (quad >= 2) s = -s;
}

// V values at p, f32 or bf16, as one access where V is 4
template <bool BF, int V>
__device__ __forceinline__ void load(const void* p, size_t at, float (&v)[V]) {
    if constexpr (BF) {
        const uint16_t* q = (const uint16_t*)p + at;
        if constexpr (V == 4) {
            const uint2 r = *(const uint2*)q;
            v[0] = __uint_as_float(r.x << 16); v[1] = __uint_as_float(r.x & 0xffff0000u);
            v[2] = __uint_as_float(r.y << 16); v[3] = __uint_as_float(r.y & 0xffff0000u);
        } else {
            v[0] = bf2f(*q);
        }
    } else {
        const float* q = (const float*)p + at;
        if constexpr (V == 4) {
            const float4 r = *(const float4*)q;
            v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w;
        } else {
            v[0] = *q;
        }
    }
}
template <bool BF, int V>
__device__ __forceinline__ void store(void* p, size_t at, const float (&v)[V]) {
    if constexpr (BF) {
        uint16_t* q = (uint16_t*)p + at;
        if constexpr (V == 4) *(uint2*)q = make_uint2(mx_bf16x2(v[0], v[1]), mx_bf16x2(v[2], v[3]));
        else *q = (uint16_t)mx_bf16x2(v[0], 0.f);
    } else {
        float* q = (float*)p + at;
        if constexpr (V == 4) *(float4*)q = make_float4(v[0], v[1], v[2], v[3]);
        else *q = v[0];
    }
}

// A unit is V pairs, or 2 V values that pass; it is the V values at `first` and the V at `second` of a head.  V = 4 where the pairs, the
// head and the rows' alignment allow it, else 1.
template <bool BI, bool BO, int V, bool NEXT>
__global__ void __launch_bounds__(kThreads) k_rope_axes(RopeArgs a) {
    const uint32_t id = blockIdx.x * kThreads + threadIdx.x;
    if (id >= a.items) return;
    const uint32_t tg = id / a.units, u = id - tg * a.units;
    const uint32_t t = tg / a.groups, g = tg - t * a.groups;
    const bool turn = u < a.turned;
    int first, second;
    float c[V], s[V];
    if (turn) {
        first = (NEXT ? 2 : 1) * V * (int)u;
        second = NEXT ? first + V : first + a.r.pairs;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int pair = V * (int)u + i;
            const int ax = a.r.axis ? min((int)a.r.axis[pair], a.r.axes - 1) : 0;
            turn_of(a.r.pos[ax * a.r.ldp + t], a.r.freq[pair], c[i], s[i]);
            c[i] *= a.r.scale;
            s[i] *= a.r.scale;
        }
    } else {
        first = 2 * a.r.pairs + 2 * V * (int)(u - a.turned);
        second = first + V;                              // V = 1: may lie past an odd head
    }
    const int h0 = (int)g * a.per, h1 = min(h0 + a.per, a.heads);
    const bool both = second < a.dim;
    for (int h = h0; h < h1; h += kBatch) {              // a batch of heads is asked for before the first of them is written
        float p[kBatch][V], q[kBatch][V];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const size_t from = (size_t)t * a.ldx + (size_t)min(h + j, h1 - 1) * a.dim;
            load<BI, V>(a.x, from + first, p[j]);
            load<BI, V>(a.x, from + (both ? second : first), q[j]);
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            if (h + j >= h1) break;
            if (turn) {
                if constexpr (NEXT && V == 4) {          // pairs (p0, p1), (p2, p3), (q0, q1), (q2, q3)
                    const float v[8] = {p[j][0], p[j][1], p[j][2], p[j][3], q[j][0], q[j][1], q[j][2], q[j][3]};
                    float w[8];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        w[2 * i] = v[2 * i] * c[i] - v[2 * i + 1] * s[i];
                        w[2 * i + 1] = v[2 * i + 1] * c[i] + v[2 * i] * s[i];
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) { p[j][i] = w[i]; q[j][i] = w[4 + i]; }
                } else {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float e = p[j][i] * c[i] - q[j][i] * s[i], f = q[j][i] * c[i] + p[j][i] * s[i];
                        p[j][i] = e;
                        q[j][i] = f;
                    }
                }
            }
            const size_t to = (size_t)t * a.ldo + (size_t)(h + j) * a.dim;
            store<BO, V>(a.out, to + first, p[j]);
            if (both) store<BO, V>(a.out, to + second, q[j]);
        }
    }
}

template <bool BI, bool BO>
void launch(const RopeArgs& a, bool vec, hipStream_t s) {
    const dim3 g((a.items + kThreads - 1) / kThreads), t(kThreads);
    if (a.r.style && vec) hipLaunchKernelGGL((k_rope_axes<BI, BO, 4, true>), g, t, 0, s, a);
    else if (a.r.style) hipLaunchKernelGGL((k_rope_axes<BI, BO, 1, true>), g, t, 0, s, a);
    else if (vec) hipLaunchKernelGGL((k_rope_axes<BI, BO, 4, false>), g, t, 0, s, a);
    else hipLaunchKernelGGL((k_rope_axes<BI, BO, 1, false>), g, t, 0, s, a);
}

}  // namespace
}  // namespace qmm

using namespace qmm;

extern "C" int qmm_rope_axes(const void* x, int dtype, size_t ldx, void* out, int out_dtype, size_t ldo, const qmm_rope* rope, int rows, int heads,
                             int dim, void* stream) {
    if ((dtype != QMM_F32 && dtype != QMM_BF16) || (out_dtype != QMM_F32 && out_dtype != QMM_BF16)) return QMM_ERR_FORMAT;
    if (!rope) return QMM_ERR_NULL;
    if (rows < 0 || heads < 1 || heads > 65536 || dim < 1 || dim > 1024) return QMM_ERR_SHAPE;
    if (rope->pairs < 0 || 2 * (int64_t)rope->pairs > dim || rope->axes < 1 || rope->axes > 255) return QMM_ERR_SHAPE;
    if (rope->style != 0 && rope->style != 1) return QMM_ERR_ARG;
    if (rows == 0) return QMM_OK;
    if (!x || !out || (rope->pairs && (!rope->freq || !rope->pos))) return QMM_ERR_NULL;
    if (ldx < (size_t)heads * dim || ldo < (size_t)heads * dim || (rope->axes > 1 && rope->ldp < (size_t)rows)) return QMM_ERR_SHAPE;
    const size_t si = dtype == QMM_BF16 ? 2 : 4, so = out_dtype == QMM_BF16 ? 2 : 4;
    if (!aligned(x, si) || !aligned(out, so) || !aligned(rope->freq, 4) || !aligned(rope->pos, 4)) return QMM_ERR_ARG;
    if (x == out && (dtype != out_dtype || ldx != ldo)) return QMM_ERR_ARG;
    RopeArgs a{x, out, *rope, ldx, ldo, 0, 0, 0, 0, heads, 0, dim};
    const bool vec = dim % 8 == 0 && rope->pairs % 4 == 0 && aligned(x, 4 * si) && aligned(out, 4 * so) && ldx % 4 == 0 && ldo % 4 == 0;
    const int V = vec ? 4 : 1;
    a.turned = (uint32_t)(rope->pairs / V);
    a.units = a.turned + (uint32_t)((dim - 2 * rope->pairs + 2 * V - 1) / (2 * V));
    // 8 heads a thread where that still leaves two waves a SIMD (2^17 threads), else fewer, down to one.  40 heads of 128 in µs, one head a
    // thread and eight: 64 tokens 3.5 and 4.5, 2048 tokens 24 and 9.5
    a.per = 8;
    while (a.per > 1 && (uint64_t)rows * ((heads + a.per - 1) / a.per) * a.units < (1u << 17)) a.per >>= 1;
    a.groups = (uint32_t)((heads + a.per - 1) / a.per);
    const uint64_t items = (uint64_t)rows * a.groups * a.units;
    if (items > 0xffffffffu - kThreads) return QMM_ERR_SHAPE;
    a.items = (uint32_t)items;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == QMM_BF16 && out_dtype == QMM_BF16) launch<true, true>(a, vec, s);
    else if (dtype == QMM_BF16) launch<true, false>(a, vec, s);
    else if (out_dtype == QMM_BF16) launch<false, true>(a, vec, s);
    else launch<false, false>(a, vec, s);
    QMM_LAUNCH_CHECK();
    return QMM_OK;
}
