// route_groups.hip -- routing with groups of experts (qmm_moe_route_groups) on gfx950, beside the plain
// top-k of moe.hip.  For a token with logits l:
//
//   s_e = softmax(l)_e or 1 / (1 + exp(-l_e)),  c_e = s_e + b_e  (b: an optional bias that balances the load)
//   value of a group = sum of its one or two largest c;  the `keep` best groups stay
//   the topk largest c of their experts, ties to the lower index;  w = s (renormalised over them) * scale
//
// Scores, sums and comparisons are in 64 bits: which of two experts is taken is a decision, and in 32 bits a
// rounding of exp could make it otherwise than the definition does.  A logit of -inf or NaN masks its expert.
//
// One wave routes a token; lane i holds the experts VPL i .. VPL i + VPL - 1, so the lowest lane of a tie has
// the lowest index.  A group's best two are found by the lanes of the group from LDS; the top-k are taken one
// at a time: the wave's largest key (the upper, then the lower half of the double's bits, by DPP), then the
// first lane that holds it.
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

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

template <int VPL>
__global__ void __launch_bounds__(256) k_route_groups(const float* __restrict__ logits, int stride, qmm_route_rule r, int* __restrict__ ids,
                                                      float* __restrict__ w, int T, int E, int topk, int lanes_per_group) {
    extern __shared__ __align__(16) double rg_lds[];     // per wave: c of every expert, the groups' values
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int t = blockIdx.x * (blockDim.x >> 6) + wave;
    if (t >= T) return;                                  // wave-uniform; no barrier below
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
        in[j] = e0 + j < E && v[j] > -INFINITY;          // false for NaN
        mx = in[j] ? fmaxf(mx, v[j]) : mx;
    }
    double p[VPL];
    if (r.score == 0) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < VPL; ++j) {                  // two infinite logits: equal, not NaN
            p[j] = in[j] ? (v[j] == mx ? 1.0 : exp((double)v[j] - (double)mx)) : 0.0;
            sum += p[j];
        }
        sum = wave_sum64(sum);
#pragma unroll
        for (int j = 0; j < VPL; ++j) p[j] /= sum;
    } else {
#pragma unroll
        for (int j = 0; j < VPL; ++j) p[j] = in[j] ? 1.0 / (1.0 + exp(-(double)v[j])) : 0.0;
    }
    double c[VPL];
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        c[j] = r.bias ? p[j] + (double)b[j] : p[j];
        in[j] = in[j] && c[j] == c[j];                   // a NaN bias masks too
    }
    const int per = E / r.groups;
    if (r.keep < r.groups) {
        double* cs = rg_lds + (size_t)wave * (E + kRgMaxGroups);
        double* gv = cs + E;
#pragma unroll
        for (int j = 0; j < VPL; ++j)
            if (e0 + j < E) cs[e0 + j] = in[j] ? c[j] : -INFINITY;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        const int g = lane / lanes_per_group, q = lane - g * lanes_per_group;
        double b1 = -INFINITY, b2 = -INFINITY;
        for (int m = q; g < r.groups && m < per; m += lanes_per_group) {
            const double x = cs[g * per + m];
            b2 = fmax(b2, fmin(b1, x));
            b1 = fmax(b1, x);
        }
        for (int o = lanes_per_group >> 1; o > 0; o >>= 1) {
            const double x1 = __shfl_xor(b1, o, 64), x2 = __shfl_xor(b2, o, 64);
            b2 = fmax(fmin(b1, x1), fmax(b2, x2));
            b1 = fmax(b1, x1);
        }
        // a group with one expert left counts that one
        const double val = r.best == 2 && b2 > -INFINITY ? b1 + b2 : b1;
        if (g < r.groups && q == 0) gv[g] = val;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        int rank = 0;
        if (lane < r.groups) {
            const double mine = gv[lane];
            for (int o = 0; o < r.groups; ++o) rank += gv[o] > mine || (gv[o] == mine && o < lane);
        }
        const uint64_t kept = __builtin_amdgcn_ballot_w64(lane < r.groups && rank < r.keep);
#pragma unroll
        for (int j = 0; j < VPL; ++j) in[j] = in[j] && (kept >> (min(e0 + j, E - 1) / per) & 1);
    }
    uint64_t key[VPL];
#pragma unroll
    for (int j = 0; j < VPL; ++j) key[j] = in[j] ? order_key(c[j]) : 0;
    double mine = 0.0, wsum = 0.0;
    int id = -1;
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
    const int slots = topk + (r.shared != 0);
    int* idt = ids + (size_t)t * slots;
    float* wt = w + (size_t)t * slots;
    if (lane < topk) {
        const double x = !r.renorm ? mine : wsum > 0.0 ? mine / wsum : 0.0;
        idt[lane] = id;
        wt[lane] = (float)(x * (double)r.scale);
    } else if (lane < slots) {
        idt[lane] = -1;
        wt[lane] = r.shared == 1 ? (float)(1.0 / (1.0 + exp(-(double)gate))) : 1.f;
    }
}

}  // namespace
}  // namespace qmm

using namespace qmm;

extern "C" int qmm_moe_route_groups(const float* logits, int stride, const qmm_route_rule* rule, int* ids, float* w, int T, int nexp, int topk,
                                    void* stream) {
    if (!logits || !rule || !ids || !w) return QMM_ERR_NULL;
    const qmm_route_rule r = *rule;
    if (r.score < 0 || r.score > 1 || r.shared < 0 || r.shared > 2 || r.best < 1 || r.best > 2) return QMM_ERR_ARG;
    if (T < 0 || nexp < 1 || nexp > kRgMaxExp || topk < 1 || topk > kRgMaxK || stride < nexp + (r.shared == 1)) return QMM_ERR_SHAPE;
    if (r.groups < 1 || r.groups > kRgMaxGroups || nexp % r.groups != 0 || r.keep < 1 || r.keep > r.groups || topk > r.keep * (nexp / r.groups))
        return QMM_ERR_SHAPE;
    if (T == 0) return QMM_OK;
    int lpg = 1;                                         // lanes that look through one group: a power of two
    while (2 * lpg * r.groups <= 64) lpg *= 2;
    // a single token: one wave; else four tokens a workgroup
    const int waves = T == 1 ? 1 : 4;
    const dim3 grid((unsigned)((T + waves - 1) / waves)), block(64 * waves);
    const size_t lds = r.keep < r.groups ? (size_t)waves * (nexp + kRgMaxGroups) * sizeof(double) : 0;
    hipStream_t s = (hipStream_t)stream;
#define QMM_RG(V) hipLaunchKernelGGL(k_route_groups<V>, grid, block, lds, s, logits, stride, r, ids, w, T, nexp, topk, lpg)
    if (nexp <= 64) QMM_RG(1);
    else if (nexp <= 128) QMM_RG(2);
    else if (nexp <= 256) QMM_RG(4);
    else if (nexp <= 512) QMM_RG(8);
    else QMM_RG(16);
#undef QMM_RG
    QMM_LAUNCH_CHECK();
    return QMM_OK;
}
