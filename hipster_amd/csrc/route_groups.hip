// route_groups.hip -- routing with groups of experts (qmm_moe_route_groups) on gfx950, beside the plain
// top-k of moe.hip.  For a token with logits l:
//
//   s_e = softmax(l)_e or 1 / (1 + exp(-l_e)),  c_e = s_e + b_e  (b: an optional bias that balances the load)
//   value of a group = sum of its one or two largest c;  the `keep` best groups stay
//   the topk largest c of their experts, ties to the lower index;  w = s (renormalised over them) * scale
//
// Scores, sums and comparisons are in 64 bits: which of two experts is taken is a decision, and in 32 bits a
// rounding of exp could make it otherwise than the definition does.  A logit or bias of -inf or NaN masks its expert.
//
// One wave routes a token; lane i holds the experts VPL i .. VPL i + VPL - 1.  The top-k without a step per expert:
// the k-th largest of the largest keys of the 32 pairs of lanes (their upper 32 bits; found by a ballot for each) is
// at most the k-th largest key, so only keys from there on are candidates, k and a few as a rule; they go to LDS in
// the experts' order, a lane each, and their rank among them is their slot.  More than 64 (many equal scores) are taken
// one at a time.
//
// 4096 tokens of 256 experts (8 groups, 4 kept, 8 chosen, sigmoid): 9.2 us (replayed), 512 of them 5.9; a single token of
// 512 (10 chosen, softmax) 5.0, 64 tokens 6.3; with a step per chosen expert, the library's exp and a branch around each 12.5
// for the first and 7.8 for the single token.  The 4 MB of logits would take 0.8: it is bound by its instructions (of a wave some
// 650 vector ones, four waves a SIMD) and, at a few tokens, by their latency.

#include "qmm_common.hpp"

namespace qmm {
namespace {

constexpr int kRgMaxExp = 1024, kRgMaxK = 16, kRgMaxGroups = 64;

__device__ __forceinline__ uint32_t readlane(uint32_t v, int l) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); }

// doubles as integers of the same order; 0 stands for a masked expert (below every real key)
__device__ __forceinline__ uint64_t order_key(double v) {
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    return b >> 63 ? ~b : b | 0x8000000000000000ull;
}

template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t umax_dpp(uint32_t v) {
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false));
}
// the wave's largest value, uniform (row_shr within 16 lanes, then row_bcast into lane 63)
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
    v = umax_dpp<0x111, 0xf>(v); v = umax_dpp<0x112, 0xf>(v); v = umax_dpp<0x114, 0xf>(v); v = umax_dpp<0x118, 0xf>(v);
    v = umax_dpp<0x142, 0xa>(v); v = umax_dpp<0x143, 0xc>(v);
    return readlane(v, 63);
}

__device__ __forceinline__ double readlane(double v, int l) {
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    return __longlong_as_double((long long)(((uint64_t)readlane((uint32_t)(b >> 32), l) << 32) | readlane((uint32_t)b, l)));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp64(double v) {      // 0.0 where no lane answers
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, ROWS, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, ROWS, 0xf, false);
    return __longlong_as_double((long long)(((uint64_t)hi << 32) | lo));
}
__device__ __forceinline__ double wave_sum64(double v) {
    v += dpp64<0x111, 0xf>(v); v += dpp64<0x112, 0xf>(v); v += dpp64<0x114, 0xf>(v); v += dpp64<0x118, 0xf>(v);
    v += dpp64<0x142, 0xa>(v); v += dpp64<0x143, 0xc>(v);
    return readlane(v, 63);
}
// v of the lane across from this one when every lane's 2 o (aligned) fold in halves: o = 1, 2, 4, 8 by DPP (the
// mirrors of 8 and 16 lanes, whose halves hold equal values by then)
__device__ __forceinline__ double fold(double v, int o) {
    switch (o) {
        case 1: return dpp64<0xb1, 0xf>(v);
        case 2: return dpp64<0x4e, 0xf>(v);
        case 4: return dpp64<0x141, 0xf>(v);
        case 8: return dpp64<0x140, 0xf>(v);
        default: return __shfl_xor(v, o, 64);
    }
}
// floats as integers of the same order
__device__ __forceinline__ uint32_t order_key32(float v) {
    const uint32_t b = __float_as_uint(v);
    return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float wave_fmax(float v) {
    const uint32_t k = wave_umax(order_key32(v));
    return __uint_as_float(k >> 31 ? k & 0x7fffffffu : ~k);
}
// exp in 64 bits: x = n ln 2 + r, the Taylor series of e^r to r^13 (|r| <= 0.347: the next term is 4e-18 of the sum) and a
// scaling by 2^n.  ln 2 is its nearest double and what is left of it: an fma rounds x - n ln 2 only once, however long
// n ln 2 is.  The products are written out: with the constant as the addend in scalar registers a term is one instruction,
// where the library's exp moves each constant first.
__device__ __forceinline__ double fma_c(double a, double b, double c) {
    double d;
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "s"(c));
    return d;
}
__device__ __forceinline__ double exp64(double x) {
    x = fmin(fmax(x, -800.0), 800.0);                    // 0 and inf from there on; a NaN becomes -800: the callers keep theirs out
    const double n = __builtin_rint(x * 1.4426950408889634);
    const double r = fma(n, -2.3190468138462996e-17, fma(n, -0.6931471805599453, x));
    double p = 1.0 / 6227020800.0;
    p = fma_c(p, r, 1.0 / 479001600.0);
    p = fma_c(p, r, 1.0 / 39916800.0);
    p = fma_c(p, r, 1.0 / 3628800.0);
    p = fma_c(p, r, 1.0 / 362880.0);
    p = fma_c(p, r, 1.0 / 40320.0);
    p = fma_c(p, r, 1.0 / 5040.0);
    p = fma_c(p, r, 1.0 / 720.0);
    p = fma_c(p, r, 1.0 / 120.0);
    p = fma_c(p, r, 1.0 / 24.0);
    p = fma_c(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return ldexp(p, (int)n);
}
constexpr int kRgCand = 64;                              // candidates: a lane each
// LDS of a wave in doubles: the choice values of the experts and the groups' values, later the candidates' keys, scores
// and experts
inline int rg_lds_doubles(int E, bool grouped) { return grouped ? (E + kRgMaxGroups > 160 ? E + kRgMaxGroups : 160) : 160; }

template <int VPL>
__global__ void __launch_bounds__(256) k_route_groups(const float* __restrict__ logits, int stride, qmm_route_rule r, int* __restrict__ ids,
                                                      float* __restrict__ w, int T, int E, int topk, int lpg_log,
                                                      uint32_t per_inv, int lds_doubles) {
    extern __shared__ __align__(16) double rg_lds[];     // per wave: c of every expert, the groups' values
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int t = blockIdx.x * (blockDim.x >> 6) + wave;
    if (t >= T) return;                                  // wave-uniform; no barrier below
    double* mem = rg_lds + (size_t)wave * lds_doubles;
    const float* l = logits + (size_t)t * stride;
    const int e0 = lane * VPL;
    float v[VPL], b[VPL];
    bool in[VPL];
#pragma unroll
    for (int j = 0; j < VPL; ++j) v[j] = l[min(e0 + j, E - 1)];
    if (r.bias) {
#pragma unroll
        for (int j = 0; j < VPL; ++j) b[j] = r.bias[min(e0 + j, E - 1)];
    }
    const float gate = r.shared == 1 ? l[E] : 0.f;
    float mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        in[j] = (e0 + j < E) & (v[j] > -INFINITY);       // false for NaN
        mx = fmaxf(mx, in[j] ? v[j] : -INFINITY);
    }
    double p[VPL];
    if (r.score == 0) {
        mx = wave_fmax(mx);
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < VPL; ++j) {                  // no branches: the exponentials run side by side
            const double x = v[j] == mx ? 0.0 : (double)v[j] - (double)mx;                   // two infinite logits: equal, not NaN
            p[j] = exp64(in[j] ? x : -800.0);
            sum += p[j];
        }
        const double inv = 1.0 / wave_sum64(sum);
#pragma unroll
        for (int j = 0; j < VPL; ++j) p[j] *= inv;
    } else {
#pragma unroll
        for (int j = 0; j < VPL; ++j) p[j] = 1.0 / (1.0 + exp64(in[j] ? -(double)v[j] : 800.0));
    }
    double c[VPL];
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        c[j] = r.bias ? p[j] + (double)b[j] : p[j];
        in[j] &= c[j] > -INFINITY;               // a bias of -inf or NaN masks too
    }
    const int per = E / r.groups;
    if (r.keep < r.groups) {
        double* cs = mem;
        const int lanes_per_group = 1 << lpg_log, g = lane >> lpg_log, q = lane & (lanes_per_group - 1);
        double b1 = -INFINITY, b2 = -INFINITY;
        auto take = [&](double v) {
            b2 = fmax(b2, fmin(b1, v));
            b1 = fmax(b1, v);
        };
        const bool own = E == 64 * VPL && lanes_per_group * r.groups == 64;
        if (own) {                                       // the lane's own experts belong to group g
#pragma unroll
            for (int j = 0; j < VPL; ++j) take(in[j] ? c[j] : -INFINITY);
        } else {
#pragma unroll
            for (int j = 0; j < VPL; ++j)
                if (e0 + j < E) cs[e0 + j] = in[j] ? c[j] : -INFINITY;
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            for (int m = q; g < r.groups && m < per; m += lanes_per_group) take(cs[g * per + m]);
        }
        for (int o = 1; o < lanes_per_group; o <<= 1) {
            const double x1 = fold(b1, o), x2 = fold(b2, o);
            b2 = fmax(fmin(b1, x1), fmax(b2, x2));
            b1 = fmax(b1, x1);
        }
        // a group with one expert left counts that one
        const double val = r.best == 2 && b2 > -INFINITY ? b1 + b2 : b1;
        int rank = 0;                                    // of the lane's group
        for (int o = 0; o < r.groups; ++o) {
            const double other = readlane(val, o * lanes_per_group);
            rank += (other > val) | ((other == val) & (o < g));
        }
        const bool stays = g < r.groups && rank < r.keep;
        const uint64_t kept = __builtin_amdgcn_ballot_w64(stays);                             // by the groups' first lanes
        // the group of expert e < 1024: e / per = e * ceil(2^20 / per) >> 20, exactly
#pragma unroll
        for (int j = 0; j < VPL; ++j)
            in[j] &= (own ? stays : (kept >> ((uint32_t)min(e0 + j, E - 1) * per_inv >> 20 << lpg_log) & 1) != 0);
    }
    uint64_t key[VPL];
#pragma unroll
    for (int j = 0; j < VPL; ++j) key[j] = in[j] ? order_key(c[j]) : 0;
    // the k-th largest of the 32 pairs of lanes' largest
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < VPL; ++j) top = max(top, (uint32_t)(key[j] >> 32));
    top = umax_dpp<0xb1, 0xf>(top);
    uint32_t least = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < 64; i += 2) {
        const uint32_t one = readlane(top, i);
        const int above = __builtin_popcountll(__builtin_amdgcn_ballot_w64(top > one));       // two lanes for each pair
        least = above < 2 * topk ? min(least, one) : least;
    }
    int n = 0, at = 0;                                   // candidates; this lane's first
    uint32_t cand = 0;
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        const bool is = (key[j] != 0) & ((uint32_t)(key[j] >> 32) >= least);
        const uint64_t m = __builtin_amdgcn_ballot_w64(is);
        n += __builtin_popcountll(m);
        at += (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
        cand |= (uint32_t)is << j;
    }
    double mine = 0.0, wsum = 0.0;
    int id = -1, slot = -1;                              // of this lane's result
    if (n <= kRgCand) {
        uint64_t* ck = (uint64_t*)mem;
        double* cp = mem + kRgCand;
        int* ce = (int*)(mem + 2 * kRgCand);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int j = 0; j < VPL; ++j)
            if (cand >> j & 1) {
                ck[at] = key[j];
                cp[at] = p[j];
                ce[at++] = e0 + j;
            }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        const uint64_t mk = lane < n ? ck[lane] : 0;
        const double mp = lane < n ? cp[lane] : 0.0;
        const int me = lane < n ? ce[lane] : -1;
        int rank = 0;
        for (int o = 0; o < n; ++o) {
            const uint64_t other = ((uint64_t)readlane((uint32_t)(mk >> 32), o) << 32) | readlane((uint32_t)mk, o);
            rank += (other > mk) | ((other == mk) & (o < lane));
        }
        if (lane < n && rank < topk) {
            slot = rank;
            id = me;
            mine = mp;
        } else if (lane >= n && lane < topk) {
            slot = lane;                                 // no expert left for it
        }
        wsum = wave_sum64(mine);
    } else {
        if (lane < topk) slot = lane;
        for (int s = 0; s < topk; ++s) {
            uint64_t head = 0;
            int hj = 0;
            double hp = 0.0;
#pragma unroll
            for (int j = 0; j < VPL; ++j) {                  // the first of the lane's largest keys
                const bool up = key[j] > head;
                head = up ? key[j] : head;
                hj = up ? j : hj;
                hp = up ? p[j] : hp;
            }
            const uint32_t hi = wave_umax((uint32_t)(head >> 32));
            const uint32_t lo = wave_umax((uint32_t)(head >> 32) == hi ? (uint32_t)head : 0u);
            if ((hi | lo) == 0) break;                       // uniform: no expert left
            const int win = __builtin_ctzll(__builtin_amdgcn_ballot_w64(head == (((uint64_t)hi << 32) | lo)));
            const uint64_t pb = (uint64_t)__double_as_longlong(hp);
            const double ps = __longlong_as_double((long long)(((uint64_t)readlane((uint32_t)(pb >> 32), win) << 32) | readlane((uint32_t)pb, win)));
            const int ej = (int)readlane((uint32_t)hj, win);
            if (lane == s) { mine = ps; id = win * VPL + ej; }
            wsum += ps;
#pragma unroll
            for (int j = 0; j < VPL; ++j) key[j] = lane == win && j == ej ? 0 : key[j];
        }
    }
    const int slots = topk + (r.shared != 0);
    int* idt = ids + (size_t)t * slots;
    float* wt = w + (size_t)t * slots;
    if (slot >= 0) {
        const double x = !r.renorm ? mine : wsum > 0.0 ? mine / wsum : 0.0;
        idt[slot] = id;
        wt[slot] = (float)(x * (double)r.scale);
    }
    if (lane == 0 && r.shared) {
        idt[topk] = -1;
        const float sig = (float)(1.0 / (1.0 + exp64(-(double)gate)));
        wt[topk] = r.shared != 1 ? 1.f : gate == gate ? sig : gate;        // a NaN stays one
    }
}

}  // namespace
}  // namespace qmm

using namespace qmm;

extern "C" int qmm_moe_route_groups(const float* logits, int stride, const qmm_route_rule* rule, int* ids, float* w, int T, int nexp, int topk,
                                    void* stream) {
    if (!rule || (T != 0 && (!logits || !ids || !w))) return QMM_ERR_NULL;
    const qmm_route_rule r = *rule;
    if (r.score < 0 || r.score > 1 || r.shared < 0 || r.shared > 2 || r.best < 1 || r.best > 2) return QMM_ERR_ARG;
    if (T < 0 || nexp < 1 || nexp > kRgMaxExp || topk < 1 || topk > kRgMaxK || stride < nexp + (r.shared == 1)) return QMM_ERR_SHAPE;
    if (r.groups < 1 || r.groups > kRgMaxGroups || nexp % r.groups != 0 || r.keep < 1 || r.keep > r.groups || topk > r.keep * (nexp / r.groups))
        return QMM_ERR_SHAPE;
    if (T == 0) return QMM_OK;
    int lpg_log = 0;                                     // lanes that look through one group: a power of two
    while ((2 << lpg_log) * r.groups <= 64) ++lpg_log;
    const int per = nexp / r.groups;
    const uint32_t per_inv = ((1u << 20) + per - 1) / per;
    // a single token: one wave; else four tokens a workgroup
    const int waves = T == 1 ? 1 : 4;
    const dim3 grid((unsigned)((T + waves - 1) / waves)), block(64 * waves);
    if (!grid_fits(grid.x, block.x)) return QMM_ERR_SHAPE;
    const int per_wave = rg_lds_doubles(nexp, r.keep < r.groups);
    const size_t lds = (size_t)waves * per_wave * sizeof(double);
    hipStream_t s = (hipStream_t)stream;
#define QMM_RG(V) hipLaunchKernelGGL(k_route_groups<V>, grid, block, lds, s, logits, stride, r, ids, w, T, nexp, topk, lpg_log, per_inv, per_wave)
    if (nexp <= 64) QMM_RG(1);
    else if (nexp <= 128) QMM_RG(2);
    else if (nexp <= 256) QMM_RG(4);
    else if (nexp <= 512) QMM_RG(8);
    else QMM_RG(16);
#undef QMM_RG
    QMM_LAUNCH_CHECK();
    return QMM_OK;
}
