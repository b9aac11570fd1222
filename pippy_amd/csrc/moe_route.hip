// Routing to experts in general form (forward and backward), and the permutation of the routed slots for many
// experts and many slots.
//
// Per token, with logits x[0 .. E):
//   score   s_e = softmax(x)_e  or  1 / (1 + exp(-x_e))
//   choice  c_e = s_e + bias_e            (bias: selection only; without one the logits rank as the scores do)
//   groups  E / n_group neighbouring experts each; the topk_group groups with the largest maximum, or the largest
//           sum of their two largest choices, stay open
//   idx     the K largest choices of open groups, descending, ties to the lower expert index
//   gate_k  = scale s[idx_k] / (renorm ? sum_j s[idx_j] : 1)
// An expert whose logit is -infinity is not there: it is never selected, and a token with fewer than K experts
// left has idx -1 and gate 0 in its last slots (pp_moe_permute drops such slots).
#include "common.h"
#include <math.h>

namespace pp {

constexpr int kRouteMaxE = 512;
constexpr int kRouteMaxK = 16;
constexpr int kRouteMaxGroups = 64;

struct RouteArgs {
    const void* logits;
    int64_t ld, T;
    const float* bias;
    int32_t E, K, n_group, topk_group;
    int32_t renorm;
    float scale;
    int32_t* idx;
    float* gate;
};

template <typename LT>
__device__ __forceinline__ float route_load(const void* p, int64_t i) {
    if constexpr (sizeof(LT) == 2) return bf16_to_f32(static_cast<const uint16_t*>(p)[i]);
    else return static_cast<const float*>(p)[i];
}

// Total order of the choices as unsigned numbers: 0 is "not there", 1 a NaN, then the numbers upwards
// (-0 counts as 0).
__device__ __forceinline__ uint64_t route_key(double c) {
    if (c != c) return 1;
    const uint64_t b = __builtin_bit_cast(uint64_t, c + 0.0);
    return (b >> 63) ? ~b : (b | (1ull << 63));
}

template <int G, typename T>
__device__ __forceinline__ T group_max(T v) {
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) {
        const T w = __shfl_xor(v, o, G);
        v = w > v ? w : v;
    }
    return v;
}
template <int G>
__device__ __forceinline__ int group_min(int v) {
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, G));
    return v;
}
template <int G, typename T>
__device__ __forceinline__ T group_sum(T v) {
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, G);
    return v;
}

// G lanes per token, V consecutive experts per lane.  Scores are formed in 64 bits: two choices that differ by
// less than an fp32 rounding are still told apart.
template <typename LT, int G, int V, bool SIGMOID, bool TOP2>
__global__ __launch_bounds__(256) void moe_route_kernel(const RouteArgs a) {
    constexpr int kTokens = 256 / G;
    __shared__ uint64_t gkey[kTokens][kRouteMaxGroups];
    __shared__ float picked[kTokens][kRouteMaxK];
    const int tid = threadIdx.x, li = tid % G, slot = tid / G;
    const int64_t t0 = (int64_t)blockIdx.x * kTokens + slot;
    const int64_t t = t0 < a.T ? t0 : a.T - 1;
    const int e0 = li * V;

    float x[V];
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        x[j] = e0 + j < a.E ? route_load<LT>(a.logits, t * a.ld + e0 + j) : -INFINITY;
        m = fmaxf(m, x[j]);
    }
    double s[V];
    if constexpr (SIGMOID) {
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] = 1.0 / (1.0 + exp(-(double)x[j]));
    } else {
        m = group_max<G>(m);
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            s[j] = x[j] == -INFINITY ? 0.0 : exp((double)x[j] - (double)m);
            sum += s[j];
        }
        sum = group_sum<G>(sum);
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] /= sum;
    }
    double c[V];
    uint64_t key[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const bool there = e0 + j < a.E && x[j] != -INFINITY;
        c[j] = a.bias && there ? s[j] + (double)a.bias[e0 + j] : s[j];
        // without a bias the logits rank exactly as the scores do, also where those saturate
        key[j] = !there ? 0 : route_key(a.bias ? c[j] : (double)x[j]);
    }
    if (a.n_group > 1) {
        const int gs = a.E / a.n_group;
        for (int g = 0; g < a.n_group; ++g) {
            uint64_t k1 = 0;
            double b1 = -INFINITY, b2 = -INFINITY;
#pragma unroll
            for (int j = 0; j < V; ++j)
                if ((e0 + j) / gs == g && key[j] > 1) {
                    if (key[j] > k1) k1 = key[j];
                    if (c[j] > b1) {
                        b2 = b1;
                        b1 = c[j];
                    } else if (c[j] > b2) {
                        b2 = c[j];
                    }
                }
            uint64_t k;
            if constexpr (TOP2) {
#pragma unroll
                for (int o = G / 2; o > 0; o >>= 1) {
                    const double o1 = __shfl_xor(b1, o, G), o2 = __shfl_xor(b2, o, G);
                    b2 = fmax(fmin(b1, o1), fmax(b2, o2));
                    b1 = fmax(b1, o1);
                }
                // a group with one expert left counts that one
                k = b1 == -INFINITY ? 0 : route_key(b2 == -INFINITY ? b1 : b1 + b2);
            } else {
                k = group_max<G>(k1);
            }
            if (li == 0) gkey[slot][g] = k;
        }
        __syncthreads();
        uint64_t open = 0;
        for (int g = 0; g < a.n_group; ++g) {
            int ahead = 0;
            for (int o = 0; o < a.n_group; ++o)
                ahead += gkey[slot][o] > gkey[slot][g] || (gkey[slot][o] == gkey[slot][g] && o < g);
            if (ahead < a.topk_group) open |= 1ull << g;
        }
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (e0 + j < a.E && !((open >> ((e0 + j) / gs)) & 1)) key[j] = 0;
    }
    for (int k = 0; k < a.K; ++k) {
        uint64_t best = key[0];
        int at = 0;
#pragma unroll
        for (int j = 1; j < V; ++j)
            if (key[j] > best) {
                best = key[j];
                at = j;
            }
        const uint64_t top = group_max<G>(best);
        const int e = group_min<G>(best == top ? e0 + at : 0x7fffffff);
        if (top != 0) {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (e0 + j == e) {
                    key[j] = 0;
                    picked[slot][k] = (float)s[j];
                }
        } else if (li == 0) {
            picked[slot][k] = 0.f;
        }
        if (li == 0 && t0 < a.T) a.idx[t * a.K + k] = top != 0 ? e : -1;
    }
    __syncthreads();
    float total = 0.f;
    for (int k = 0; k < a.K; ++k) total += picked[slot][k];
    const float f = a.renorm ? (total == 0.f ? 0.f : a.scale / total) : a.scale;
    if (t0 < a.T)
        for (int k = li; k < a.K; k += G) a.gate[t * a.K + k] = picked[slot][k] * f;
}

// ---- backward -----------------------------------------------------------------------------------
// With g'_k = s[idx_k] / S, S = sum_j s[idx_j]:
//   d s[idx_k] = scale (dgate_k - sum_j g'_j dgate_j) / S   (renorm),   scale dgate_k   (otherwise)
//   softmax: dx_e = s_e (ds_e - sum_j s_j ds_j);   sigmoid: dx_e = ds_e s_e (1 - s_e)
// dgate_k is given, or <dout[t], y[pos(t, k)]> over the expert rows.  One wave per token.
struct RouteBwdArgs {
    const void* logits;
    int64_t ld, T;
    int32_t E, K, renorm;
    float scale;
    const int32_t* idx;
    const float* dgate;
    const uint16_t* dout; int64_t ld_dout;
    const uint16_t* y; int64_t ld_y;
    const int32_t* pos;
    int32_t C8;
    void* dlogits;
    int64_t ld_dl;
    int32_t cols;  // columns E .. cols-1 of dlogits become zeros
};

template <typename LT, bool SIGMOID>
__global__ __launch_bounds__(256) void moe_route_bwd_kernel(const RouteBwdArgs a) {
    constexpr int V = kRouteMaxE / 64;
    const int lane = threadIdx.x & 63;
    const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= a.T) return;
    float x[V];
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int e = j * 64 + lane;
        x[j] = e < a.E ? route_load<LT>(a.logits, t * a.ld + e) : -INFINITY;
        m = fmaxf(m, x[j]);
    }
    float s[V];
    if constexpr (SIGMOID) {
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] = 1.0f / (1.0f + expf(-x[j]));
    } else {
        m = wave_max(m);
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            s[j] = x[j] == -INFINITY ? 0.f : expf(x[j] - m);
            sum += s[j];
        }
        sum = wave_sum(sum);
        const float inv = sum == 0.f ? 0.f : 1.0f / sum;  // no expert is there: no score, no gradient
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] *= inv;
    }
    // the slots of this token: gradient of the weight and the score, in every lane
    float dg[kRouteMaxK], sk[kRouteMaxK];
    float total = 0.f;
#pragma unroll
    for (int k = 0; k < kRouteMaxK; ++k) {
        dg[k] = sk[k] = 0.f;
        if (k >= a.K) break;
        const int e = a.idx[t * a.K + k];
        if (e < 0 || e >= a.E) continue;
        if (a.dgate) {
            dg[k] = a.dgate[t * a.K + k];
        } else {
            const int r = a.pos[t * a.K + k];
            if (r >= 0) {
                float d = 0.f;
                const uint4* yp = reinterpret_cast<const uint4*>(a.y + (int64_t)r * a.ld_y);
                const uint4* op = reinterpret_cast<const uint4*>(a.dout + t * a.ld_dout);
                for (int c = lane; c < a.C8; c += 64) {
                    const uint4 u = yp[c], v = op[c];
                    d = fmaf(bf16lo(u.x), bf16lo(v.x), d); d = fmaf(bf16hi(u.x), bf16hi(v.x), d);
                    d = fmaf(bf16lo(u.y), bf16lo(v.y), d); d = fmaf(bf16hi(u.y), bf16hi(v.y), d);
                    d = fmaf(bf16lo(u.z), bf16lo(v.z), d); d = fmaf(bf16hi(u.z), bf16hi(v.z), d);
                    d = fmaf(bf16lo(u.w), bf16lo(v.w), d); d = fmaf(bf16hi(u.w), bf16hi(v.w), d);
                }
                dg[k] = wave_sum(d);
            }
        }
        float own = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (j * 64 + lane == e) own = s[j];
        sk[k] = __shfl(own, e & 63, 64);
        total += sk[k];
    }
    // With renorm the differences are taken against the first slot's gradient (the weights sum to one): a token
    // with a single expert gets exactly no gradient.  Then sum_j s_j ds_j is zero, and softmax scores pass
    // nothing on to the experts that were not selected.
    float dot = 0.f;  // sum_j s_j ds_j over the selected experts
    float along = 0.f;
    if (a.renorm) {
        const float ref = dg[0];
#pragma unroll
        for (int k = 0; k < kRouteMaxK; ++k) {
            if (k >= a.K) break;
            dg[k] -= ref;
            along = fmaf(sk[k], dg[k], along);
        }
    }
#pragma unroll
    for (int k = 0; k < kRouteMaxK; ++k) {
        if (k >= a.K) break;
        if (a.renorm) {
            dg[k] = total == 0.f ? 0.f : a.scale * (dg[k] - along / total) / total;
        } else {
            dg[k] *= a.scale;
            dot = fmaf(sk[k], dg[k], dot);
        }
    }
    float d[V];
#pragma unroll
    for (int j = 0; j < V; ++j) d[j] = 0.f;
#pragma unroll
    for (int k = 0; k < kRouteMaxK; ++k) {
        if (k >= a.K) break;
        const int e = a.idx[t * a.K + k];
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (j * 64 + lane == e) d[j] += dg[k];
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int e = j * 64 + lane;
        if (e >= a.cols) continue;
        float dx = 0.f;
        if (e < a.E) dx = SIGMOID ? d[j] * s[j] * (1.0f - s[j]) : s[j] * (d[j] - dot);
        if constexpr (sizeof(LT) == 2) static_cast<uint16_t*>(a.dlogits)[t * a.ld_dl + e] = f32_to_bf16(dx);
        else static_cast<float*>(a.dlogits)[t * a.ld_dl + e] = dx;
    }
}

// ---- permutation --------------------------------------------------------------------------------
// A stable counting sort by expert.  A work-group takes kPermSlots consecutive slots, a wave a consecutive part
// of them.  First launch: the counts of every work-group.  Second launch: every work-group adds up the counts
// in front of it, ranks its slots in order and places them.  A wave finds the lanes that hold the same expert
// from one ballot per bit of the expert index; the first of them does the counting for all.
constexpr int kPermMaxE = 1024;
constexpr int kPermThreads = 256;
constexpr int kPermSlots = 2048;
constexpr int kPermWaves = kPermThreads / 64;

__device__ __forceinline__ unsigned long long same_expert(int e, int bits) {
    unsigned long long m = __ballot(e >= 0);
    for (int b = 0; b < bits; ++b) {
        const unsigned long long set = __ballot((e >> b) & 1);
        m &= ((e >> b) & 1) ? set : ~set;
    }
    return m;
}

__device__ __forceinline__ int perm_expert(const int32_t* ids, int64_t i, int64_t n, int E) {
    const int e = i < n ? ids[i] : -1;
    return e >= 0 && e < E ? e : -1;
}

// Orders a wave's LDS accesses with those of its other lanes.
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Counts of this work-group's waves into cnt[wave][E].
__device__ __forceinline__ void perm_count(int (*cnt)[kPermMaxE], const int32_t* ids, int64_t n, int E, int bits) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int i = tid; i < kPermWaves * kPermMaxE; i += kPermThreads) (&cnt[0][0])[i] = 0;
    __syncthreads();
    const int64_t first = (int64_t)blockIdx.x * kPermSlots + wave * (kPermSlots / kPermWaves);
    for (int q = 0; q < kPermSlots / kPermWaves; q += 64) {
        const int e = perm_expert(ids, first + q + lane, n, E);
        const unsigned long long m = same_expert(e, bits);
        if (e >= 0 && __ffsll(m) - 1 == lane) cnt[wave][e] += __popcll(m);
        wave_lds_fence();
    }
    __syncthreads();
}

__global__ __launch_bounds__(kPermThreads) void moe_permute_count_kernel(const int32_t* __restrict__ ids, int64_t n,
                                                                         int E, int bits, int32_t* __restrict__ ws) {
    __shared__ int cnt[kPermWaves][kPermMaxE];
    perm_count(cnt, ids, n, E, bits);
    for (int e = threadIdx.x; e < E; e += kPermThreads) {
        int s = 0;
        for (int w = 0; w < kPermWaves; ++w) s += cnt[w][e];
        ws[(int64_t)blockIdx.x * E + e] = s;
    }
}

__global__ __launch_bounds__(kPermThreads) void moe_permute_place_kernel(const int32_t* __restrict__ ids, int64_t n,
                                                                         int E, int bits, const int32_t* __restrict__ ws,
                                                                         int32_t* __restrict__ seg_start,
                                                                         int32_t* __restrict__ row_src,
                                                                         int32_t* __restrict__ pos) {
    __shared__ int cnt[kPermWaves][kPermMaxE];
    __shared__ int sum[kPermThreads];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    perm_count(cnt, ids, n, E, bits);
    // per expert (4 consecutive ones per thread): its total, and what lies in front of this work-group
    constexpr int V = kPermMaxE / kPermThreads;
    int total[V], before[V], mine = 0;
    for (int j = 0; j < V; ++j) {
        const int e = tid * V + j;
        total[j] = before[j] = 0;
        if (e < E)
            for (unsigned b = 0; b < gridDim.x; ++b) {
                const int v = ws[(int64_t)b * E + e];
                total[j] += v;
                if (b < blockIdx.x) before[j] += v;
            }
        mine += total[j];
    }
    sum[tid] = mine;
    __syncthreads();
    for (int o = 1; o < kPermThreads; o <<= 1) {
        const int add = tid >= o ? sum[tid - o] : 0;
        __syncthreads();
        sum[tid] += add;
        __syncthreads();
    }
    int begin = sum[tid] - mine;
    for (int j = 0; j < V; ++j) {
        const int e = tid * V + j;
        if (e < E) {
            if (blockIdx.x == 0) seg_start[e] = begin;
            int at = begin + before[j];  // the waves of this work-group, one after the other
            for (int w = 0; w < kPermWaves; ++w) {
                const int v = cnt[w][e];
                cnt[w][e] = at;
                at += v;
            }
        }
        begin += total[j];
    }
    if (blockIdx.x == 0 && tid == kPermThreads - 1) seg_start[E] = sum[tid];
    __syncthreads();
    const int64_t first = (int64_t)blockIdx.x * kPermSlots + wave * (kPermSlots / kPermWaves);
    for (int q = 0; q < kPermSlots / kPermWaves; q += 64) {
        const int64_t i = first + q + lane;
        const int e = perm_expert(ids, i, n, E);
        const unsigned long long m = same_expert(e, bits);
        int r = -1;
        if (e >= 0) r = cnt[wave][e] + __popcll(m & ((1ull << lane) - 1ull));
        // every lane has read before the first lane of a set writes, and that is written before the next round
        wave_lds_fence();
        if (e >= 0 && __ffsll(m) - 1 == lane) cnt[wave][e] = r + __popcll(m);
        wave_lds_fence();
        if (i < n) {
            pos[i] = r;
            if (r >= 0) row_src[r] = (int)i;
        }
    }
}

static int64_t perm_groups(int64_t n) { return n > 0 ? (n + kPermSlots - 1) / kPermSlots : 1; }

template <typename LT, bool SIGMOID, bool TOP2>
static int route_launch(const RouteArgs& a, hipStream_t st) {
    auto go = [&](auto kernel, int tokens) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)((a.T + tokens - 1) / tokens)), dim3(256), 0, st, a);
        return check_launch("moe_route_kernel");
    };
    if (a.E <= 16) return go(moe_route_kernel<LT, 8, 2, SIGMOID, TOP2>, 32);
    if (a.E <= 64) return go(moe_route_kernel<LT, 16, 4, SIGMOID, TOP2>, 16);
    if (a.E <= 256) return go(moe_route_kernel<LT, 32, 8, SIGMOID, TOP2>, 8);
    return go(moe_route_kernel<LT, 64, 8, SIGMOID, TOP2>, 4);
}

static int route_check(const char* who, const pp_moe_route_desc* d) {
    if (!d) return fail(PP_ERR_INVALID, "%s: null descriptor", who);
    if (d->T < 0 || d->T > 0x7fffffff || d->E < 2 || d->E > kRouteMaxE || d->topk < 1 || d->topk > kRouteMaxK ||
        d->topk > d->E || d->ld < d->E)
        return fail(PP_ERR_INVALID, "%s: bad shape (T=%lld E=%d topk=%d ld=%lld; 2 to %d experts, at most %d per token)",
                    who, (long long)d->T, d->E, d->topk, (long long)d->ld, kRouteMaxE, kRouteMaxK);
    if (d->scoring != PP_MOE_SOFTMAX && d->scoring != PP_MOE_SIGMOID)
        return fail(PP_ERR_INVALID, "%s: unknown scoring %d", who, d->scoring);
    if (d->dtype != PP_BF16 && d->dtype != PP_F32) return fail(PP_ERR_INVALID, "%s: unknown dtype %d", who, d->dtype);
    if (!d->logits || !d->topk_idx) return fail(PP_ERR_INVALID, "%s: null pointer", who);
    if (!(d->scale == d->scale) || d->scale == INFINITY || d->scale == -INFINITY)
        return fail(PP_ERR_INVALID, "%s: scale must be finite", who);
    return PP_OK;
}

}  // namespace pp

using namespace pp;

extern "C" int pp_moe_route(const pp_moe_route_desc* d, pp_stream stream) {
    const int rc = route_check("pp_moe_route", d);
    if (rc) return rc;
    const int ng = d->n_group > 1 ? d->n_group : 1, kg = ng > 1 ? d->topk_group : 1;
    if (ng > kRouteMaxGroups || d->E % ng || kg < 1 || kg > ng || d->topk > d->E / ng * kg ||
        (d->group_score != PP_MOE_GROUP_MAX && d->group_score != PP_MOE_GROUP_TOP2))
        return fail(PP_ERR_INVALID, "pp_moe_route: bad groups (%d of %d groups of %d experts for %d slots; at most %d groups)",
                    d->topk_group, d->n_group, d->E, d->topk, kRouteMaxGroups);
    if (!d->gate) return fail(PP_ERR_INVALID, "pp_moe_route: null pointer");
    if (d->T == 0) return PP_OK;
    RouteArgs a;
    a.logits = d->logits; a.ld = d->ld; a.T = d->T; a.bias = d->bias;
    a.E = d->E; a.K = d->topk; a.n_group = ng; a.topk_group = kg;
    a.renorm = d->renorm; a.scale = d->scale; a.idx = d->topk_idx; a.gate = d->gate;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const bool sig = d->scoring == PP_MOE_SIGMOID, top2 = d->group_score == PP_MOE_GROUP_TOP2;
    if (d->dtype == PP_BF16) {
        if (sig) return top2 ? route_launch<uint16_t, true, true>(a, st) : route_launch<uint16_t, true, false>(a, st);
        return top2 ? route_launch<uint16_t, false, true>(a, st) : route_launch<uint16_t, false, false>(a, st);
    }
    if (sig) return top2 ? route_launch<float, true, true>(a, st) : route_launch<float, true, false>(a, st);
    return top2 ? route_launch<float, false, true>(a, st) : route_launch<float, false, false>(a, st);
}

extern "C" int pp_moe_route_bwd(const pp_moe_route_desc* d, pp_stream stream) {
    const int rc = route_check("pp_moe_route_bwd", d);
    if (rc) return rc;
    if (!d->dlogits || d->cols_dl < d->E || d->cols_dl > kRouteMaxE || d->ld_dl < d->cols_dl)
        return fail(PP_ERR_INVALID, "pp_moe_route_bwd: bad dlogits (cols=%d ld=%lld for %d experts)", d->cols_dl,
                    (long long)d->ld_dl, d->E);
    if (!d->dgate) {
        if (!d->dout || !d->y || !d->pos || d->C < 8 || d->C % 8 || d->C > (1 << 24) || d->ld_dout % 8 || d->ld_y % 8 ||
            d->ld_dout < d->C || d->ld_y < d->C || !aligned(d->dout, 16) || !aligned(d->y, 16))
            return fail(PP_ERR_INVALID, "pp_moe_route_bwd: needs dgate, or dout, y and pos (16-byte aligned, widths and "
                        "leading dimensions multiples of 8; C=%lld)", (long long)d->C);
    }
    if (d->T == 0) return PP_OK;
    RouteBwdArgs a;
    a.logits = d->logits; a.ld = d->ld; a.T = d->T; a.E = d->E; a.K = d->topk; a.renorm = d->renorm; a.scale = d->scale;
    a.idx = d->topk_idx; a.dgate = d->dgate;
    a.dout = static_cast<const uint16_t*>(d->dout); a.ld_dout = d->ld_dout;
    a.y = static_cast<const uint16_t*>(d->y); a.ld_y = d->ld_y;
    a.pos = d->pos; a.C8 = (int32_t)(d->C / 8);
    a.dlogits = d->dlogits; a.ld_dl = d->ld_dl; a.cols = d->cols_dl;
    hipStream_t st = static_cast<hipStream_t>(stream);
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)((a.T + 3) / 4)), dim3(256), 0, st, a);
        return check_launch("moe_route_bwd_kernel");
    };
    const bool sig = d->scoring == PP_MOE_SIGMOID;
    if (d->dtype == PP_BF16) return sig ? go(moe_route_bwd_kernel<uint16_t, true>) : go(moe_route_bwd_kernel<uint16_t, false>);
    return sig ? go(moe_route_bwd_kernel<float, true>) : go(moe_route_bwd_kernel<float, false>);
}

extern "C" int64_t pp_moe_permute_workspace_ints(int64_t n_slots, int E) {
    if (n_slots < 0 || n_slots > 0x7fffffff || E < 1 || E > kPermMaxE) return -1;
    return perm_groups(n_slots) * E;
}

extern "C" int pp_moe_permute_ws(const int32_t* expert_of_slot, int64_t n_slots, int E, int32_t* seg_start,
                                 int32_t* row_src, int32_t* pos, int32_t* workspace, int64_t workspace_ints,
                                 pp_stream stream) {
    const int64_t need = pp_moe_permute_workspace_ints(n_slots, E);
    if (need < 0 || !seg_start || (n_slots > 0 && (!expert_of_slot || !row_src || !pos)))
        return fail(PP_ERR_INVALID, "pp_moe_permute_ws: bad arguments (n_slots=%lld E=%d, at most %d experts)",
                    (long long)n_slots, E, kPermMaxE);
    if (!workspace || workspace_ints < need)
        return fail(PP_ERR_INVALID, "pp_moe_permute_ws: workspace of %lld ints, needs %lld", (long long)workspace_ints,
                    (long long)need);
    int bits = 0;
    while ((1 << bits) < E) ++bits;
    const dim3 grid((unsigned)perm_groups(n_slots));
    hipStream_t st = static_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(moe_permute_count_kernel, grid, dim3(kPermThreads), 0, st, expert_of_slot, n_slots, E, bits, workspace);
    int rc = check_launch("moe_permute_count_kernel");
    if (rc) return rc;
    hipLaunchKernelGGL(moe_permute_place_kernel, grid, dim3(kPermThreads), 0, st, expert_of_slot, n_slots, E, bits, workspace,
                       seg_start, row_src, pos);
    return check_launch("moe_permute_place_kernel");
}
