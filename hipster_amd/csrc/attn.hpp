// attn.hpp -- what the kernels of attention share: a call's sequences, a paged MXFP4 cache, bf16 matrix instructions.
#pragma once
#include "mx.hpp"

namespace qmm {

typedef __bf16 at_bf2 __attribute__((ext_vector_type(2)));
typedef __bf16 at_bf8 __attribute__((ext_vector_type(8)));
typedef short at_s4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kMxNan = 253;                         // scale bytes from here on: 255 is NaN, 253 and 254 hold values that bf16 does not
constexpr float kLog2e = 1.44269504088896340736f;
__device__ __forceinline__ float neg_inf() { return __uint_as_float(0xff800000u); }

// other lanes of the wave read what this one wrote to LDS (which the hardware does in order), or write what it read
__device__ __forceinline__ void wave_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local"); }

// The transposing LDS read of 16-bit values: in each 16 lanes, lane i supplies the address of four values, values 4 (i % 4) .. + 3 of
// row i / 4, and gets value i of the four rows.
__device__ __forceinline__ at_s4 tr_read(const void* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) at_s4*)(const __attribute__((address_space(3))) at_s4*)p);
}

// ---- a call's sequences (qmm_seqs) ----
// Offsets and lengths are device data.  Both ends of a span are brought into [0, rows] before they are subtracted (a difference of
// arbitrary ints wraps round), so that whatever they hold, rows r0 .. r0 + m - 1 are rows; positions are checked by the callers.
__host__ __device__ __forceinline__ int within(int v, int rows) { return v < 0 ? 0 : v > rows ? rows : v; }
struct SeqSpan { int r0, m, len; };               // first row, rows, tokens

__device__ __forceinline__ SeqSpan seq_span(const int* __restrict__ cu, const int* __restrict__ lens, int b, int rows) {
    const int r0 = within(cu[b], rows), r1 = within(cu[b + 1], rows);
    return {r0, max(r1 - r0, 0), max(lens[b], 0)};
}

// the sum of the lanes up to this one: within rows of 16 lanes by shifts, then the rows' last sums to the rows behind them
__device__ __forceinline__ uint32_t wave_upto(uint32_t v) {
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false);       // from 1, 2, 4, 8 lanes below
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false);       // lane 15 of the row below, rows 1 and 3
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false);       // lane 31, rows 2 and 3
    return v;
}

// The sequence that row r (the same in all lanes) belongs to and its span, -1: none.  The wave looks at 64 sequences at a time, so that
// up to 64 cost one load's latency.
__device__ __forceinline__ int seq_of_row(const int* __restrict__ cu, const int* __restrict__ lens, int n, int rows, int r, SeqSpan& q) {
    const int lane = threadIdx.x & 63;
    int b = -1, from = 0, to = 0, len = 0;               // of the last sequence that begins at r or before it
    for (int base = 0; base < n; base += 64) {
        const int at = base + lane;
        int c0 = 0x7fffffff, c1 = 0, c2 = 0;
        if (at < n) { c0 = cu[at]; c1 = cu[at + 1]; c2 = lens[at]; }
        const int below = __popcll(__ballot(at < n && c0 <= r));
        if (below) {
            const int l = below - 1;
            b = base + l;
            from = __builtin_amdgcn_readlane(c0, l);
            to = __builtin_amdgcn_readlane(c1, l);
            len = __builtin_amdgcn_readlane(c2, l);
        }
        if (below < 64) break;
    }
    b = __builtin_amdgcn_readfirstlane(b);
    if (b < 0 || r >= to || r < from) return -1;
    const int r0 = within(from, rows);
    q = {r0, max(within(to, rows) - r0, 0), max(len, 0)};
    return b;
}

// ---- softmax, in powers of two ----
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

inline bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// what the entry points ask of a cache and of the sequences; *lg: log2 of the page
inline int kv_check(const qmm_kv_mxfp4* kv, const qmm_seqs* s, int* lg) {
    if (!kv || !s || !kv->kq || !kv->ke || !kv->vq || !kv->ve || !s->cu || !s->lens || !s->table) return QMM_ERR_NULL;
    if (kv->dim != 64 && kv->dim != 128 && kv->dim != 256) return QMM_ERR_SHAPE;
    if (kv->heads < 1 || kv->heads > 4096 || kv->pages < 1 || kv->page < 16 || kv->page > 4096 || (kv->page & (kv->page - 1))) return QMM_ERR_SHAPE;
    if (s->n < 1 || s->ld < 1 || (int64_t)s->ld * kv->page > 0x7fffffff) return QMM_ERR_SHAPE;
    if (!aligned(kv->kq, 16) || !aligned(kv->vq, 16) || !aligned(kv->ke, 8) || !aligned(kv->ve, 8)) return QMM_ERR_ARG;
    if (!aligned(s->cu, 4) || !aligned(s->lens, 4) || !aligned(s->table, 4)) return QMM_ERR_ARG;
    for (*lg = 4; 1 << *lg != kv->page;) ++*lg;
    return QMM_OK;
}
inline int attn_check(const qmm_attn* a) {
    if (!a) return QMM_ERR_NULL;
    if (a->window < 0) return QMM_ERR_SHAPE;
    if (!(a->scale >= -0x1p100f && a->scale <= 0x1p100f)) return QMM_ERR_ARG;          // times log2(e) it is finite; NaN
    return aligned(a->sinks, 4) ? QMM_OK : QMM_ERR_ARG;
}

}  // namespace qmm
