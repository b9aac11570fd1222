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
constexpr int kRouteList = 64;  // entries of the list that the experts are selected from

struct RouteArgs {
    const void* logits;
    int64_t ld, T;
    const float* bias;
    int32_t E, K, n_group, topk_group;
    int32_t group_top2, renorm;
    int32_t vec, vec_bias;  // rows of logits, the bias are 16-byte aligned
    float scale;
    int32_t* idx;
    float* gate;
};
constexpr float kRouteLog2e = 1.44269504088896340736f;

// Orders a wave's LDS accesses with those of its other lanes.
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

template <typename LT>
__device__ __forceinline__ float route_load(const void* p, int64_t i) {
    if constexpr (sizeof(LT) == 2) return bf16_to_f32(static_cast<const uint16_t*>(p)[i]);
    else return static_cast<const float*>(p)[i];
}

// Total order as unsigned numbers: 0 is "not there", 1 a NaN, then the numbers upwards (-0 counts as 0).
__device__ __forceinline__ uint32_t route_key(float c) {
    if (c != c) return 1;
    const uint32_t b = __float_as_uint(c + 0.0f);
    return (b >> 31) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float route_value(uint32_t key) {  // of a key > 1
    return __uint_as_float((key >> 31) ? key & 0x7fffffffu : ~key);
}

// Reductions over the G neighbouring lanes of a token; every lane gets the result.  Inside 16 lanes the partners come
// through DPP (two quad permutations and two mirrors; after a step all lanes of a set hold the same), beyond that
// through a shuffle.
template <int CTRL>
__device__ __forceinline__ uint32_t route_dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
template <int G, typename F>
__device__ __forceinline__ uint32_t route_reduce(uint32_t v, F f) {
    static_assert(G == 8 || G == 16 || G == 32, "lanes per token");
    v = f(v, route_dpp<0xB1>(v));   // quad_perm 1 0 3 2
    v = f(v, route_dpp<0x4E>(v));   // quad_perm 2 3 0 1
    v = f(v, route_dpp<0x141>(v));  // row_half_mirror
    if constexpr (G >= 16) v = f(v, route_dpp<0x140>(v));  // row_mirror
    if constexpr (G >= 32) v = f(v, (uint32_t)__shfl_xor((int)v, 16, 64));
    return v;
}
template <int G>
__device__ __forceinline__ uint32_t route_max(uint32_t v) {
    return route_reduce<G>(v, [](uint32_t x, uint32_t y) { return x > y ? x : y; });
}
template <int G>
__device__ __forceinline__ uint32_t route_min(uint32_t v) {
    return route_reduce<G>(v, [](uint32_t x, uint32_t y) { return x < y ? x : y; });
}
template <int G>
__device__ __forceinline__ float route_fmax(float v) {
    return __uint_as_float(route_reduce<G>(__float_as_uint(v), [](uint32_t x, uint32_t y) {
        return __float_as_uint(fmaxf(__uint_as_float(x), __uint_as_float(y)));
    }));
}
template <int G>
__device__ __forceinline__ float route_fsum(float v) {
    return __uint_as_float(route_reduce<G>(__float_as_uint(v), [](uint32_t x, uint32_t y) {
        return __float_as_uint(__uint_as_float(x) + __uint_as_float(y));
    }));
}

// Sigmoid scores for the weights: e^-ref / (1 + e^-x), with both exponents at most 0.  Renormalised weights take them relative
// to the largest selected logit where that is negative: fp32 holds no score below e^-103, but their ratios it does.
__device__ __forceinline__ float route_sigmoid(float x, float ref) { return expf(fminf(x, 0.f) - ref) / (1.0f + expf(-fabsf(x))); }
// The largest logit whose score 64 bits hold as 0 (e^-x overflows): selected logits that are all as low, as a mask writes
// them, have a sum of 0 and weights of 0.
constexpr float kRouteNoScore = -709.78271484375f;
__device__ __forceinline__ float route_sigmoid_renorm(float x, float most) {
    return most <= kRouteNoScore && x == x ? 0.f : route_sigmoid(x, fminf(most, 0.f));
}

// How far apart two choices formed in fp32 must be for their order to be certain.  A score is off by at most
//   sigmoid: s (1 - s) (1.5 |x| 2^-24 + 2^-23) from the exponential (|x| s (1 - s) < 0.23), 3 s 2^-24 from the quotient:
//            below 2^-21;
//   softmax: s (|x - m| 2^-24 + 2^-23) from the exponential (|x - m| s < 0.37 s_max), s (V + 5 + 4) 2^-24 from the sum and
//            the quotient: below 2^-19 of the row's largest score for V <= 16;
// and the sum with the bias by half a step of itself.  The margin is twice that.
template <bool SIGMOID>
__device__ __forceinline__ float route_margin(float s_max, float c) {
    return (SIGMOID ? 0x1p-20f : 0x1p-18f * s_max) + 0x1p-22f * fabsf(c);
}

// The same values in 64 bits, for the few experts whose order fp32 leaves open.
template <bool SIGMOID>
__device__ __forceinline__ double route_score64(float x, float m, double sum) {
    if constexpr (SIGMOID) return 1.0 / (1.0 + exp(-(double)x));
    else return (x == m ? 1.0 : exp((double)x - (double)m)) / sum;
}
template <typename LT, int G>
__device__ __forceinline__ double route_sum64(const RouteArgs& a, int64_t t, int li, float m) {
    double sum = 0.0;
    for (int e = li; e < a.E; e += G) {
        const float x = route_load<LT>(a.logits, t * a.ld + e);
        if (x == x && x != -INFINITY) sum += x == m ? 1.0 : exp((double)x - (double)m);
    }
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    return sum;
}

// G lanes per token, V consecutive experts per lane, V <= 16.  Without a bias the keys are the logits, exact, and
// equal ones go to the lowest index.  With one they are the fp32 choices; experts within the margin of one that is
// selected (a token in a thousand) are compared in 64 bits.  The weights are formed from the selected experts'
// logits alone.
//
// The selection is K rounds of: largest key of the lanes, the experts that may hold it, the winner; or, for more than
// 64 experts and K > 4, ranks inside a short list, whose cost hardly grows with K.  us, rounds | list, 8192 tokens,
// without a bias: E = 64, K = 4: 4.4 | 4.8, 8: 5.6 | 5.6, 16: 7.8 | 14.2 (so 8 lanes have no list); E = 128, K = 4: 4.9 | 5.2,
// 6: 5.6 | 5.3, 16: 9.5 | 6.6; E = 256, K = 8: 8.2 | 6.3; E = 512, K = 8: 12.6 | 8.0, 16: 19.2 | 9.0.  With a bias E = 256, K = 8:
// 11.2 | 8.8, in 8 groups, 4 of them kept: 13.2 | 9.4 to 11.7 (8.9 MB: 1.8 us of memory
// time; the same with no choice left to 64 bits as with the usual one in a thousand).
// Bound by instructions (a round is about 5 V + 30 for 64 / G tokens a wave) and, below a few thousand tokens, by
// latency (16 experts with K = 2 take 3.4 us).  16 lanes of 16 experts for E = 256 make a round four tokens' worth of
// work per wave; a wave per token spends most of a round on the reductions.
template <typename LT, int G, int V, bool SIGMOID, bool BIASED>
__global__ __launch_bounds__(256) void moe_route_kernel(const RouteArgs a) {
    constexpr int kTokens = 256 / G, kE = G * V;
    __shared__ __attribute__((aligned(16))) uint32_t gkey[kTokens][kRouteMaxGroups];
    __shared__ double wide[kTokens][kRouteMaxGroups];
    __shared__ int chosen[kTokens][kRouteMaxK];
    // the keys of the group scores, later the list
    constexpr bool kListed = G >= 16;
    constexpr int kWords = kE < 2 * G ? 2 * G : kE;
    static_assert(!kListed || (kWords >= 2 * kRouteList && kRouteList <= kRouteMaxGroups), "rows of shared memory");
    __shared__ __attribute__((aligned(16))) uint32_t words[kTokens][kWords];
    auto& ckey = words;
    auto list = reinterpret_cast<uint64_t (*)[kWords / 2]>(&words[0][0]);
    __shared__ int listed[kTokens];
    const int tid = threadIdx.x, li = tid % G, slot = tid / G, lane = tid & 63;
    const int64_t t0 = (int64_t)blockIdx.x * kTokens + slot;
    const int64_t t = t0 < a.T ? t0 : a.T - 1;
    const int e0 = li * V;
    const unsigned long long mine = ((1ull << (G & 63)) - 1ull) << (lane & ~(G - 1));  // this token's lanes

    float x[V];
    constexpr int kVec = 16 / (int)sizeof(LT);
    bool done = false;
    if constexpr (V % kVec == 0) {
        if (a.vec && e0 + V <= a.E) {
            const uint4* p = reinterpret_cast<const uint4*>(static_cast<const LT*>(a.logits) + t * a.ld + e0);
#pragma unroll
            for (int i = 0; i < V / kVec; ++i) {
                const uint4 w = p[i];
                const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    if constexpr (sizeof(LT) == 2) {
                        x[i * 8 + 2 * q] = bf16lo(u[q]);
                        x[i * 8 + 2 * q + 1] = bf16hi(u[q]);
                    } else {
                        x[i * 4 + q] = __uint_as_float(u[q]);
                    }
                }
            }
            done = true;
        }
    }
    if (!done) {
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = e0 + j < a.E ? route_load<LT>(a.logits, t * a.ld + e0 + j) : -INFINITY;
    }

    // scores of all experts in fp32, where anything needs them: the choices of a bias or of sums over groups, or
    // the sum of softmax weights that are not renormalised
    const bool top2 = a.n_group > 1 && a.group_top2;
    // (a NaN enters neither the maximum nor the sum of the choices, only its own; infinite logits share all of the softmax)
    float m = -INFINITY, sum = 1.f, s_max = 1.f;
    float s[V];
#pragma unroll
    for (int j = 0; j < V; ++j) s[j] = 0.f;
    if constexpr (SIGMOID) {
        if (BIASED || top2) {
#pragma unroll
            for (int j = 0; j < V; ++j) s[j] = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-x[j] * kRouteLog2e));
        }
    } else if (BIASED || top2 || !a.renorm) {
#pragma unroll
        for (int j = 0; j < V; ++j) m = fmaxf(m, x[j]);
        m = route_fmax<G>(m);
        sum = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            s[j] = x[j] == -INFINITY ? 0.f : expf(x[j] - m);
            sum += s[j];
        }
        sum = route_fsum<G>(sum);
        const bool lost = sum != sum;  // the row has a NaN or an infinite logit
        if (__any(lost)) {
            float known = 0.f;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if (lost) s[j] = x[j] == -INFINITY ? 0.f : x[j] == m ? 1.f : expf(x[j] - m);
                known += x[j] == x[j] ? s[j] : 0.f;
            }
            known = route_fsum<G>(known);
            if (lost) sum = known;
        }
        s_max = 1.0f / sum;
        if (lost && !a.renorm) sum = NAN;  // such a row's softmax weights
        if (BIASED || top2) {
#pragma unroll
            for (int j = 0; j < V; ++j) s[j] *= s_max;
        }
    }
    uint32_t key[V];
    float bias[BIASED ? V : 1];
    if constexpr (BIASED) {
        if (V % 4 == 0 && a.vec_bias && e0 + V <= a.E) {
#pragma unroll
            for (int i = 0; i < V / 4; ++i) {
                const float4 w = reinterpret_cast<const float4*>(a.bias + e0)[i];
                bias[4 * i] = w.x; bias[4 * i + 1] = w.y; bias[4 * i + 2] = w.z; bias[4 * i + 3] = w.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) bias[j] = e0 + j < a.E ? a.bias[e0 + j] : 0.f;
        }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const bool there = e0 + j < a.E && x[j] != -INFINITY;
        if constexpr (BIASED) key[j] = there ? route_key(s[j] + bias[j]) : 0;
        else key[j] = there ? route_key(x[j]) : 0;
    }

    if (a.n_group > 1) {
        const int gs = a.E / a.n_group;
        const bool summed = top2;
        // What the group scores are made of: a maximum ranks as the keys do, sums need the choices themselves.
        // Where every lane's experts belong to one group the lane hands on its two largest, else all of them.
        const bool own_group = gs % V == 0;
        const int parts = own_group ? gs / V : gs;  // entries per group
        if (own_group) {
            uint32_t k1 = 0, k2 = 0;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const uint32_t k = key[j] == 0 ? 0 : (summed && !BIASED ? route_key(s[j]) : key[j]);
                const uint32_t lo = k < k1 ? k : k1;
                k1 = k > k1 ? k : k1;
                k2 = lo > k2 ? lo : k2;
            }
            ckey[slot][li] = k1;
            ckey[slot][G + li] = k2;
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                ckey[slot][e0 + j] = key[j] == 0 ? 0 : (summed && !BIASED ? route_key(s[j]) : key[j]);
        }
        wave_lds_fence();
        const int n_mine = (a.n_group - li + G - 1) / G;  // groups li, li + G, ... are this lane's
        unsigned long long open = 0;
        uint32_t kept_min = 0xffffffffu, shut_max = 0;
        for (int q = 0; q < n_mine; ++q) {
            const int g = li + q * G;
            uint32_t k1 = 0, k2 = 0;
            for (int i = g * parts; i < (g + 1) * parts; ++i) {
                const uint32_t k = ckey[slot][i];
                const uint32_t lo = k < k1 ? k : k1;
                k1 = k > k1 ? k : k1;
                k2 = lo > k2 ? lo : k2;
                if (own_group) {
                    const uint32_t second = ckey[slot][G + i];
                    k2 = second > k2 ? second : k2;
                }
            }
            // a group with one expert left counts that one; a NaN counts as not there
            gkey[slot][g] = !summed ? (k1 > 1 ? k1 : 0) : k1 <= 1 ? 0 : k2 <= 1 ? k1 : route_key(route_value(k1) + route_value(k2));
        }
        wave_lds_fence();
        for (int q = 0; q * G < a.n_group; ++q) {
            const int g = li + q * G;
            const uint32_t own = g < a.n_group ? gkey[slot][g] : 0;
            int ahead = 0;
#pragma unroll 8
            for (int o = 0; o < a.n_group; ++o) {
                const uint32_t other = gkey[slot][o];
                ahead += other > own || (other == own && o < g);
            }
            const bool kept = g < a.n_group && ahead < a.topk_group;
            open |= ((__ballot(kept) & mine) >> (lane & ~(G - 1))) << (q * G);
            if (kept) kept_min = own < kept_min ? own : kept_min;
            else if (g < a.n_group) shut_max = own > shut_max ? own : shut_max;
        }
        // group scores in fp32 whose order is open, at the border: again in 64 bits, from the members that may be
        // the largest (each member is off by half a margin, the sum of two by one)
        if (BIASED || summed) {
            kept_min = route_min<G>(kept_min);
            shut_max = route_max<G>(shut_max);
            bool doubt = false;
            if (shut_max > 1 && kept_min > 1) {
                const float hi = route_value(kept_min), lo = route_value(shut_max);
                doubt = hi - lo <= 2.0f * route_margin<SIGMOID>(s_max, fmaxf(fabsf(hi), fabsf(lo)));
            }
            if (__any(doubt)) {
                const double total = SIGMOID ? 1.0 : route_sum64<LT, G>(a, t, li, m);
                wave_lds_fence();
#pragma unroll
                for (int j = 0; j < V; ++j)
                    ckey[slot][e0 + j] = key[j] == 0 ? 0 : (summed && !BIASED ? route_key(s[j]) : key[j]);
                wave_lds_fence();
                const float border = route_value(kept_min), beyond = route_value(shut_max);
                const float apart = 2.0f * route_margin<SIGMOID>(s_max, fmaxf(fabsf(border), fabsf(beyond)));
                for (int q = 0; q < n_mine; ++q) {
                    const int g = li + q * G;
                    // far from the border: certain either way
                    const float own = route_value(gkey[slot][g]);
                    if (gkey[slot][g] <= 1 || own < border - apart || own > beyond + apart) {
                        wide[slot][g] = gkey[slot][g] > 1 && own > beyond + apart ? INFINITY : -INFINITY;
                        continue;
                    }
                    uint32_t k1 = 0, k2 = 0;
#pragma unroll 8
                    for (int e = g * gs; e < (g + 1) * gs; ++e) {
                        const uint32_t k = ckey[slot][e];
                        const uint32_t lo = k < k1 ? k : k1;
                        k1 = k > k1 ? k : k1;
                        k2 = lo > k2 ? lo : k2;
                    }
                    double b1 = -INFINITY, b2 = -INFINITY;
                    if (k1 > 1) {
                        const float v = route_value(summed && k2 > 1 ? k2 : k1);
                        const uint32_t from = route_key(v - route_margin<SIGMOID>(s_max, v));
                        for (int first = g * gs, left = gs; left > 0; first += 32, left -= 32) {
                            uint32_t may = 0;
#pragma unroll 8
                            for (int i = 0; i < (left < 32 ? left : 32); ++i) {
                                const uint32_t k = ckey[slot][first + i];
                                may |= (k > 1 && k >= from ? 1u : 0u) << i;
                            }
                            for (; may; may &= may - 1) {
                                const int e = first + __ffs(may) - 1;
                                double c = route_score64<SIGMOID>(route_load<LT>(a.logits, t * a.ld + e), m, total);
                                if constexpr (BIASED) c += (double)a.bias[e];
                                if (c > b1) {
                                    b2 = b1;
                                    b1 = c;
                                } else if (c > b2) {
                                    b2 = c;
                                }
                            }
                        }
                    }
                    wide[slot][g] = !summed || b2 == -INFINITY ? b1 : b1 + b2;
                }
                wave_lds_fence();
                unsigned long long again = 0;
                for (int q = 0; q * G < a.n_group; ++q) {
                    const int g = li + q * G;
                    const double own = g < a.n_group ? wide[slot][g] : 0.0;
                    int ahead = 0;
#pragma unroll 8
                    for (int o = 0; o < a.n_group; ++o) {
                        const double other = wide[slot][o];
                        ahead += other > own || (other == own && o < g);
                    }
                    again |= ((__ballot(g < a.n_group && ahead < a.topk_group) & mine) >> (lane & ~(G - 1))) << (q * G);
                }
                if (doubt) open = again;
            }
        }
        int g = e0 / gs, left = (g + 1) * gs - e0;  // group of the expert, experts up to its end
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (e0 + j < a.E && !((open >> g) & 1)) key[j] = 0;
            if (--left == 0) {
                ++g;
                left = gs;
            }
        }
    }

    // From a short list: whatever is selected is at least as large as the K-th largest of the lanes' (for 16 lanes, of
    // their halves') largest keys.  Every expert on the list counts the ones ahead of it, all at once.  A list that
    // is too long (a row in ascending order, equal logits) is left to the rounds.
    bool rounds = !kListed || a.K <= 4;
    if (kListed && !rounds) {
        constexpr int S = G == 16 ? 2 : 1;
        uint32_t top[S];
#pragma unroll
        for (int h = 0; h < S; ++h) {
            top[h] = key[h * (V / S)];
#pragma unroll
            for (int j = 1; j < V / S; ++j) top[h] = key[h * (V / S) + j] > top[h] ? key[h * (V / S) + j] : top[h];
            gkey[slot][S * li + h] = top[h];
        }
        if (li == 0) listed[slot] = 0;
#pragma unroll
        for (int q = 0; q < (kRouteMaxK + G - 1) / G; ++q)
            if (li + q * G < a.K) chosen[slot][li + q * G] = -1;
        wave_lds_fence();
        uint32_t from = 0xffffffffu;
        int ahead[S] = {};
#pragma unroll
        for (int o = 0; o < S * G; o += 4) {
            const uint4 w = *reinterpret_cast<const uint4*>(&gkey[slot][o]);
#pragma unroll
            for (int h = 0; h < S; ++h) ahead[h] += (w.x > top[h]) + (w.y > top[h]) + (w.z > top[h]) + (w.w > top[h]);
        }
#pragma unroll
        for (int h = 0; h < S; ++h)
            if (ahead[h] < a.K) from = top[h] < from ? top[h] : from;
        from = route_min<G>(from);
        if constexpr (BIASED) {
            if (from > 1) {
                const float v = route_value(from);
                from = route_key(v - route_margin<SIGMOID>(s_max, v));
            }
        }
        from = from < 1 ? 1 : from;
        int mine_listed = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) mine_listed += key[j] >= from;
        int at = mine_listed ? atomicAdd(&listed[slot], mine_listed) : 0;  // (any order: ranks do not depend on it)
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (key[j] < from) continue;
            if (at < kRouteList) list[slot][at] = (uint64_t)key[j] << 32 | (uint32_t)(0xffff - (e0 + j));
            ++at;
        }
        wave_lds_fence();
        const int n = listed[slot];
        rounds = n > kRouteList;
        bool doubt = false;
        if (!rounds) {
            for (int i = li; i < n; i += G) {
                const uint64_t own = list[slot][i];
                uint32_t near_from = 0;
                if constexpr (BIASED) {
                    const float v = route_value((uint32_t)(own >> 32));
                    near_from = route_key(v - route_margin<SIGMOID>(s_max, v));
                }
                int before = 0, near = 0;
#pragma unroll 4
                for (int o = 0; o < n; ++o) {
                    const uint64_t other = list[slot][o];
                    before += other > own;
                    if constexpr (BIASED) near += (uint32_t)(other >> 32) >= near_from;
                }
                if (before < a.K) {
                    chosen[slot][before] = 0xffff - (int)(uint32_t)own;
                    // one behind it, and within the margin
                    if (BIASED && (own >> 32) > 1 && near > before + 1) doubt = true;
                }
            }
        }
        if constexpr (BIASED) {
            doubt = (__ballot(doubt) & mine) != 0;
            if (__any(doubt)) {
                const double total = SIGMOID ? 1.0 : route_sum64<LT, G>(a, t, li, m);
                if (doubt) {
                    for (int i = li; i < n; i += G) {
                        const int e = 0xffff - (int)(uint32_t)list[slot][i];
                        wide[slot][i] = route_score64<SIGMOID>(route_load<LT>(a.logits, t * a.ld + e), m, total) + (double)a.bias[e];
                    }
                }
                wave_lds_fence();
                if (doubt) {
                    for (int i = li; i < n; i += G) {
                        const double own = wide[slot][i];
                        const int e = 0xffff - (int)(uint32_t)list[slot][i];
                        int before = 0;
#pragma unroll 4
                        for (int o = 0; o < n; ++o) {
                            const double other = wide[slot][o];
                            const bool lower = 0xffff - (int)(uint32_t)list[slot][o] < e;
                            before += other > own || (other == own && lower) || (own != own && (other == other || lower));
                        }
                        if (before < a.K) chosen[slot][before] = e;
                    }
                }
            }
        }
    }
    if (__any(rounds))
    for (int k = 0; k < a.K; ++k) {
        uint32_t best = key[0];
#pragma unroll
        for (int j = 1; j < V; ++j) best = key[j] > best ? key[j] : best;
        const uint32_t top = route_max<G>(best);
        uint32_t from = top;
        if constexpr (BIASED) {
            if (top > 1) {
                const float v = route_value(top);
                from = route_key(v - route_margin<SIGMOID>(s_max, v));
                from = from < 2 ? 2 : from;  // (a NaN is no candidate beside a number)
            }
        }
        uint32_t cand = 0;  // this lane's experts that may be the largest
#pragma unroll
        for (int j = 0; j < V; ++j) cand |= (key[j] >= from ? 1u : 0u) << j;
        if (top == 0 || !rounds) cand = 0;
        int at = __ffs(cand) - 1;
        unsigned long long holders = __ballot(cand != 0) & mine;
        if constexpr (BIASED) {
            const bool several = (cand & (cand - 1)) != 0 || (cand != 0 && (holders & (holders - 1)) != 0);
            if (__any(several && top > 1)) {
                const double total = SIGMOID ? 1.0 : route_sum64<LT, G>(a, t, li, m);
                double c = -INFINITY;
                for (uint32_t left = top > 1 ? cand : 0; left; left &= left - 1) {
                    const int j = __ffs(left) - 1;
                    float xj = x[0], bj = bias[0];
#pragma unroll
                    for (int i = 1; i < V; ++i) {
                        xj = i == j ? x[i] : xj;
                        bj = i == j ? bias[i] : bj;
                    }
                    const double w = route_score64<SIGMOID>(xj, m, total) + (double)bj;
                    if (w > c) {
                        c = w;
                        at = j;
                    }
                }
                double most = c;
#pragma unroll
                for (int o = G / 2; o > 0; o >>= 1) most = fmax(most, __shfl_xor(most, o, 64));
                const unsigned long long wide_holders = __ballot(cand != 0 && (top <= 1 || c == most)) & mine;
                if (top > 1) holders = wide_holders;
            }
        }
        const bool winner = cand != 0 && __ffsll(holders) - 1 == lane;
        if (winner) {
#pragma unroll
            for (int j = 0; j < V; ++j) key[j] = j == at ? 0 : key[j];
            chosen[slot][k] = e0 + at;
        }
        if (top == 0 && rounds && li == 0) chosen[slot][k] = -1;
    }
    wave_lds_fence();

    // the weights of the selected experts; kRouteMaxK / G slots per lane at most
    constexpr int kOwn = (kRouteMaxK + G - 1) / G;
    int e[kOwn];
    float w[kOwn], xs[kOwn], part = 0.f, most = -INFINITY;
#pragma unroll
    for (int q = 0; q < kOwn; ++q) {
        const int k = li + q * G;
        e[q] = k < a.K ? chosen[slot][k] : -1;
        xs[q] = e[q] >= 0 ? route_load<LT>(a.logits, t * a.ld + e[q]) : -INFINITY;
        most = fmaxf(most, xs[q]);
    }
    // renormalised weights need no other expert: relative to the largest selected logit
    if (a.renorm) most = route_fmax<G>(most);
#pragma unroll
    for (int q = 0; q < kOwn; ++q) {
        if (SIGMOID) w[q] = a.renorm ? route_sigmoid_renorm(xs[q], most) : route_sigmoid(xs[q], 0.f);
        else w[q] = a.renorm ? expf(xs[q] - most) : expf(xs[q] - m) / sum;
        if (e[q] < 0) w[q] = 0.f;
        part += w[q];
    }
    const float total = route_fsum<G>(part);
#pragma unroll
    for (int q = 0; q < kOwn; ++q) {
        const int k = li + q * G;
        if (k >= a.K || t0 >= a.T) continue;
        a.idx[t * a.K + k] = e[q];
        // (a token of no expert, or of scores that are all 0)
        a.gate[t * a.K + k] = e[q] < 0 || (a.renorm && total == 0.f) ? 0.f : a.renorm ? a.scale * (w[q] / total) : a.scale * w[q];
    }
}

// ---- backward -----------------------------------------------------------------------------------
// With g'_k = s[idx_k] / sum_j s[idx_j]:
//   d s[idx_k] = scale (dgate_k - sum_j g'_j dgate_j) / sum_j s[idx_j]   (renorm),   scale dgate_k   (otherwise)
//   softmax: dx_e = s_e (ds_e - sum_j s_j ds_j);   sigmoid: dx_e = ds_e s_e (1 - s_e)
// Renormalised softmax weights are a softmax over the selected logits alone, dx_k = scale g'_k (dgate_k - sum g' dgate),
// sigmoid ones have a factor (1 - s_k) besides (formed from the weights g', not from ds, whose quotient overflows where all
// scores are small), and sigmoid scores do not mix: only softmax weights that are not renormalised read the whole row.
// dgate_k is given, or <dout[t], y[pos(t, k)]> over the expert rows.
//
// One wave per token; lane k < K holds slot k.  Bound by the expert rows: per chunk of 512 columns the loads of the
// gradient row and of all K expert rows go out together.  [4093 tokens, 6 of 64 experts, 1024 columns]: 13.2 us, 4.5
// TB/s over 59 MB.
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

__device__ __forceinline__ float route_dot8(const uint4& u, const uint4& v, float d) {
    d = fmaf(bf16lo(u.x), bf16lo(v.x), d); d = fmaf(bf16hi(u.x), bf16hi(v.x), d);
    d = fmaf(bf16lo(u.y), bf16lo(v.y), d); d = fmaf(bf16hi(u.y), bf16hi(v.y), d);
    d = fmaf(bf16lo(u.z), bf16lo(v.z), d); d = fmaf(bf16hi(u.z), bf16hi(v.z), d);
    d = fmaf(bf16lo(u.w), bf16lo(v.w), d); d = fmaf(bf16hi(u.w), bf16hi(v.w), d);
    return d;
}

// KM: slots rounded up to a power of two
template <typename LT, bool SIGMOID, int KM>
__global__ __launch_bounds__(256) void moe_route_bwd_kernel(const RouteBwdArgs a) {
    constexpr int V = kRouteMaxE / 64;
    __shared__ float row[4][kRouteMaxE];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t t = (int64_t)blockIdx.x * 4 + wave;
    if (t >= a.T) return;  // (no work-group barrier below)
    const bool slot = lane < a.K;
    int e = slot ? a.idx[t * a.K + lane] : -1;
    if (e >= a.E) e = -1;
    const float xe = e >= 0 ? route_load<LT>(a.logits, t * a.ld + e) : -INFINITY;

    float dg = 0.f;  // gradient of this lane's slot
    if (a.dgate) {
        if (e >= 0) dg = a.dgate[t * a.K + lane];
    } else {
        const int pos = slot && e >= 0 ? a.pos[t * a.K + lane] : -1;
        const uint4* rows[KM];
        float acc[KM];
        bool there[KM];
#pragma unroll
        for (int k = 0; k < KM; ++k) {
            const int r = __builtin_amdgcn_readlane(pos, k);
            there[k] = r >= 0;
            rows[k] = reinterpret_cast<const uint4*>(a.y + (int64_t)(r >= 0 ? r : 0) * a.ld_y);
            acc[k] = 0.f;
        }
        const uint4* op = reinterpret_cast<const uint4*>(a.dout + t * a.ld_dout);
        for (int c = lane; c < a.C8; c += 64) {
            const uint4 v = op[c];
            uint4 u[KM];
#pragma unroll
            for (int k = 0; k < KM; ++k)
                if (there[k]) u[k] = rows[k][c];
#pragma unroll
            for (int k = 0; k < KM; ++k)
                if (there[k]) acc[k] = route_dot8(u[k], v, acc[k]);
        }
#pragma unroll
        for (int k = 0; k < KM; ++k) {
            const float d = wave_sum(acc[k]);
            if (lane == k && there[k]) dg = d;
        }
    }

    float s[V], dx;
    float dot = 0.f;
    if (SIGMOID || a.renorm) {
        float w;
        const float most = a.renorm ? wave_max(xe) : 0.f;
        if constexpr (SIGMOID) w = a.renorm ? route_sigmoid_renorm(xe, most) : route_sigmoid(xe, 0.f);
        else w = expf(xe - most);
        if (e < 0) w = 0.f;
        float ds = a.scale * dg;
        if (a.renorm) {
            // differences against the first slot's gradient (the weights sum to one): a token with a single expert
            // gets exactly no gradient
            const float total = wave_sum(w), g = total == 0.f ? 0.f : w / total;
            const float rel = dg - __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(dg)));
            ds = a.scale * (rel - wave_sum(e >= 0 ? g * rel : 0.f));
            dx = ds * g;
            if (SIGMOID) dx *= route_sigmoid(-xe, 0.f);  // 1 - s, which a subtraction would lose for large logits
        } else {
            dx = ds * w * route_sigmoid(-xe, 0.f);
        }
        if (e < 0) dx = 0.f;
    } else {
        float x[V], m = -INFINITY;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = j * 64 + lane;
            x[j] = c < a.E ? route_load<LT>(a.logits, t * a.ld + c) : -INFINITY;
            m = fmaxf(m, x[j]);
        }
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
        const float ds = e >= 0 ? a.scale * dg : 0.f, w = e >= 0 ? expf(xe - m) * inv : 0.f;
        dot = wave_sum(e >= 0 ? w * ds : 0.f);
        dx = ds;
    }
    // slots of one expert add up (in slot order), then the row goes out
    float mine = 0.f;
#pragma unroll
    for (int k = 0; k < KM; ++k) {
        const int ek = __builtin_amdgcn_readlane(e, k);
        const float dk = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(dx), k));
        if (ek == e) mine += dk;
    }
    for (int c = lane; c < a.E; c += 64) row[wave][c] = 0.f;
    wave_lds_fence();
    if (e >= 0) row[wave][e] = mine;
    wave_lds_fence();
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = j * 64 + lane;
        if (c >= a.cols) break;
        float v = c < a.E ? row[wave][c] : 0.f;
        if (!SIGMOID && !a.renorm) v = c < a.E ? s[j] * (v - dot) : 0.f;
        if constexpr (sizeof(LT) == 2) static_cast<uint16_t*>(a.dlogits)[t * a.ld_dl + c] = f32_to_bf16(v);
        else static_cast<float*>(a.dlogits)[t * a.ld_dl + c] = v;
    }
}

// ---- permutation --------------------------------------------------------------------------------
// A stable counting sort by expert.  A work-group takes 1024 ROUNDS consecutive slots, a wave a consecutive part of
// them, 64 at a time: one ballot per bit of the expert index gives every lane the set of lanes that hold its
// expert; its rank is the wave's count so far plus the members in front of it, and the first member counts for all.
// Up to 4096 slots are one launch of one work-group.  More are two: the counts of every work-group, then every
// work-group adds up the counts of all and of those in front of it and places its slots.  More rounds mean fewer
// work-groups and fewer counts to read but longer chains; us for 1, 2, 4, 8 rounds, 256 experts: 65536 slots 8.8, 9.4, 12.8,
// 21.4; 131072: 10.7, 10.4, 13.2, 20.0; 262144: 15.0, 12.8, 14.5, 20.7; 393216: 21.0, 15.1, 15.9, 21.6; 524288: 25.2, 17.6, 17.3,
// 22.5; 1048576: 68, 30, 23, 26; 1310720: 115, 52, 32, 28 (64 experts: 65536 9.3, 9.3; 524288: 20.0, 14.4, 14.5; 1048576: 54, 24,
// 19, 22).
constexpr int kPermMaxE = 1024;
constexpr int kPermThreads = 1024;
constexpr int kPermWaves = kPermThreads / 64;
constexpr int kPermOneLaunch = 4 * kPermThreads;
constexpr int64_t kPermMaxSlots = 1 << 24;

__device__ __forceinline__ unsigned long long same_expert(int e, int bits) {
    unsigned long long m = __ballot(e >= 0);
    for (int b = 0; b < bits; ++b) {
        const unsigned long long set = __ballot((e >> b) & 1);
        m &= ((e >> b) & 1) ? set : ~set;
    }
    return m;
}

// Ranks this work-group's slots inside their wave: e[q] the expert of the lane's q-th slot (-1: none), r[q] its rank;
// cnt[wave][E] the wave's counts.
template <int ROUNDS>
__device__ __forceinline__ void perm_rank(int (*cnt)[kPermMaxE], const int32_t* ids, int64_t n, int E, int bits,
                                          int (&e)[ROUNDS], int (&r)[ROUNDS]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t first = (int64_t)blockIdx.x * (ROUNDS * kPermThreads) + wave * (64 * ROUNDS) + lane;
#pragma unroll
    for (int q = 0; q < ROUNDS; ++q) {
        e[q] = first + q * 64 < n ? ids[first + q * 64] : -1;
        if (e[q] >= E) e[q] = -1;
    }
    for (int i = lane; i < E; i += 64) cnt[wave][i] = 0;
    wave_lds_fence();
#pragma unroll
    for (int q = 0; q < ROUNDS; ++q) {
        const unsigned long long m = same_expert(e[q], bits);
        r[q] = 0;
        if (e[q] >= 0) r[q] = cnt[wave][e[q]] + __popcll(m & ((1ull << lane) - 1ull));
        // every lane has read before the first lane of a set writes, and that is written before the next round
        wave_lds_fence();
        if (e[q] >= 0 && __ffsll(m) - 1 == lane) cnt[wave][e[q]] = r[q] + __popcll(m);
        wave_lds_fence();
    }
    __syncthreads();
}

template <int ROUNDS>
__global__ __launch_bounds__(kPermThreads) void moe_permute_count_kernel(const int32_t* __restrict__ ids, int64_t n,
                                                                         int E, int bits, int32_t* __restrict__ ws) {
    __shared__ int cnt[kPermWaves][kPermMaxE];
    int e[ROUNDS], r[ROUNDS];
    perm_rank(cnt, ids, n, E, bits, e, r);
    if ((int)threadIdx.x < E) {
        int s = 0;
#pragma unroll
        for (int w = 0; w < kPermWaves; ++w) s += cnt[w][threadIdx.x];
        ws[(int64_t)blockIdx.x * E + threadIdx.x] = s;
    }
}

template <int ROUNDS>
__global__ __launch_bounds__(kPermThreads) void moe_permute_place_kernel(const int32_t* __restrict__ ids, int64_t n,
                                                                         int E, int bits, const int32_t* __restrict__ ws,
                                                                         int32_t* __restrict__ seg_start,
                                                                         int32_t* __restrict__ row_src,
                                                                         int32_t* __restrict__ pos) {
    __shared__ int cnt[kPermWaves][kPermMaxE];
    __shared__ int wave_total[kPermWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int e[ROUNDS], r[ROUNDS];
    perm_rank(cnt, ids, n, E, bits, e, r);
    // expert tid: its total over all work-groups, and what lies in front of this one
    int total = 0, before = 0;
    if (tid < E) {
        if (gridDim.x == 1) {
#pragma unroll
            for (int w = 0; w < kPermWaves; ++w) total += cnt[w][tid];
        } else {
#pragma unroll 16
            for (unsigned b = 0; b < gridDim.x; ++b) {
                const int v = ws[(int64_t)b * E + tid];
                total += v;
                before += b < blockIdx.x ? v : 0;
            }
        }
    }
    int upto = total;  // running sum over the experts: inside the wave, then over the waves
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int add = __shfl_up(upto, o, 64);
        if (lane >= o) upto += add;
    }
    if (lane == 63) wave_total[wave] = upto;
    __syncthreads();
    for (int w = 0; w < wave; ++w) upto += wave_total[w];
    if (tid < E) {
        const int begin = upto - total;
        if (blockIdx.x == 0) {
            seg_start[tid] = begin;
            if (tid == E - 1) seg_start[E] = upto;
        }
        int at = begin + before;  // the waves of this work-group, one after the other
#pragma unroll
        for (int w = 0; w < kPermWaves; ++w) {
            const int v = cnt[w][tid];
            cnt[w][tid] = at;
            at += v;
        }
    }
    __syncthreads();
    const int64_t first = (int64_t)blockIdx.x * (ROUNDS * kPermThreads) + wave * (64 * ROUNDS) + lane;
#pragma unroll
    for (int q = 0; q < ROUNDS; ++q) {
        const int64_t i = first + q * 64;
        if (i >= n) continue;
        const int at = e[q] >= 0 ? cnt[wave][e[q]] + r[q] : -1;
        pos[i] = at;
        if (at >= 0) row_src[at] = (int)i;
    }
}

// The rounds that measured fastest (above).
static int perm_rounds(int64_t n) {
    if (n <= kPermOneLaunch) return 4;
    return n <= 1 << 16 ? 1 : n <= 1 << 19 ? 2 : n <= 1 << 20 ? 4 : 8;
}
static int64_t perm_groups(int64_t n) {
    const int64_t slots = (int64_t)perm_rounds(n) * kPermThreads;
    return n > 0 ? (n + slots - 1) / slots : 1;
}

template <int ROUNDS>
static int perm_launch(const int32_t* ids, int64_t n, int E, int32_t* seg_start, int32_t* row_src, int32_t* pos,
                       int32_t* ws, hipStream_t st) {
    int bits = 0;
    while ((1 << bits) < E) ++bits;
    const dim3 grid((unsigned)perm_groups(n));
    if (grid.x > 1) {
        hipLaunchKernelGGL(moe_permute_count_kernel<ROUNDS>, grid, dim3(kPermThreads), 0, st, ids, n, E, bits, ws);
        const int rc = check_launch("moe_permute_count_kernel");
        if (rc) return rc;
    }
    hipLaunchKernelGGL(moe_permute_place_kernel<ROUNDS>, grid, dim3(kPermThreads), 0, st, ids, n, E, bits, ws, seg_start,
                       row_src, pos);
    return check_launch("moe_permute_place_kernel");
}

template <typename LT, bool SIGMOID, bool BIASED>
static int route_launch(const RouteArgs& a, hipStream_t st) {
    auto go = [&](auto kernel, int tokens) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)((a.T + tokens - 1) / tokens)), dim3(256), 0, st, a);
        return check_launch("moe_route_kernel");
    };
    if (a.E <= 16) return go(moe_route_kernel<LT, 8, 2, SIGMOID, BIASED>, 32);
    if (a.E <= 64) return go(moe_route_kernel<LT, 8, 8, SIGMOID, BIASED>, 32);
    if (a.E <= 128) return go(moe_route_kernel<LT, 16, 8, SIGMOID, BIASED>, 16);
    if (a.E <= 256) return go(moe_route_kernel<LT, 16, 16, SIGMOID, BIASED>, 16);
    return go(moe_route_kernel<LT, 32, 16, SIGMOID, BIASED>, 8);
}

template <typename LT, bool SIGMOID>
static int route_bwd_launch(const RouteBwdArgs& a, hipStream_t st) {
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)((a.T + 3) / 4)), dim3(256), 0, st, a);
        return check_launch("moe_route_bwd_kernel");
    };
    if (a.K <= 2) return go(moe_route_bwd_kernel<LT, SIGMOID, 2>);
    if (a.K <= 4) return go(moe_route_bwd_kernel<LT, SIGMOID, 4>);
    if (a.K <= 8) return go(moe_route_bwd_kernel<LT, SIGMOID, 8>);
    return go(moe_route_bwd_kernel<LT, SIGMOID, 16>);
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
    if (d->T > 0 && (!d->logits || !d->topk_idx)) return fail(PP_ERR_INVALID, "%s: null pointer", who);
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
    if (d->T == 0) return PP_OK;  // (empty tensors have no address)
    if (!d->gate) return fail(PP_ERR_INVALID, "pp_moe_route: null pointer");
    RouteArgs a;
    a.logits = d->logits; a.ld = d->ld; a.T = d->T; a.bias = d->bias;
    a.E = d->E; a.K = d->topk; a.n_group = ng; a.topk_group = kg;
    a.renorm = d->renorm; a.scale = d->scale; a.idx = d->topk_idx; a.gate = d->gate;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int64_t size = d->dtype == PP_BF16 ? 2 : 4;
    a.group_top2 = d->group_score == PP_MOE_GROUP_TOP2;
    a.vec = aligned(d->logits, 16) && d->ld * size % 16 == 0;
    a.vec_bias = aligned(d->bias, 16);
    const bool sig = d->scoring == PP_MOE_SIGMOID, biased = d->bias != nullptr;
    if (d->dtype == PP_BF16) {
        if (sig) return biased ? route_launch<uint16_t, true, true>(a, st) : route_launch<uint16_t, true, false>(a, st);
        return biased ? route_launch<uint16_t, false, true>(a, st) : route_launch<uint16_t, false, false>(a, st);
    }
    if (sig) return biased ? route_launch<float, true, true>(a, st) : route_launch<float, true, false>(a, st);
    return biased ? route_launch<float, false, true>(a, st) : route_launch<float, false, false>(a, st);
}

extern "C" int pp_moe_route_bwd(const pp_moe_route_desc* d, pp_stream stream) {
    const int rc = route_check("pp_moe_route_bwd", d);
    if (rc) return rc;
    if (d->T == 0) return PP_OK;
    if (!d->dlogits || d->cols_dl < d->E || d->cols_dl > kRouteMaxE || d->ld_dl < d->cols_dl)
        return fail(PP_ERR_INVALID, "pp_moe_route_bwd: bad dlogits (cols=%d ld=%lld for %d experts)", d->cols_dl,
                    (long long)d->ld_dl, d->E);
    if (!d->dgate) {
        if (!d->dout || !d->y || !d->pos || d->C < 8 || d->C % 8 || d->C > (1 << 24) || d->ld_dout % 8 || d->ld_y % 8 ||
            d->ld_dout < d->C || d->ld_y < d->C || !aligned(d->dout, 16) || !aligned(d->y, 16))
            return fail(PP_ERR_INVALID, "pp_moe_route_bwd: needs dgate, or dout, y and pos (16-byte aligned, widths and "
                        "leading dimensions multiples of 8; C=%lld)", (long long)d->C);
    }
    RouteBwdArgs a;
    a.logits = d->logits; a.ld = d->ld; a.T = d->T; a.E = d->E; a.K = d->topk; a.renorm = d->renorm; a.scale = d->scale;
    a.idx = d->topk_idx; a.dgate = d->dgate;
    a.dout = static_cast<const uint16_t*>(d->dout); a.ld_dout = d->ld_dout;
    a.y = static_cast<const uint16_t*>(d->y); a.ld_y = d->ld_y;
    a.pos = d->pos; a.C8 = (int32_t)(d->C / 8);
    a.dlogits = d->dlogits; a.ld_dl = d->ld_dl; a.cols = d->cols_dl;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const bool sig = d->scoring == PP_MOE_SIGMOID;
    if (d->dtype == PP_BF16) return sig ? route_bwd_launch<uint16_t, true>(a, st) : route_bwd_launch<uint16_t, false>(a, st);
    return sig ? route_bwd_launch<float, true>(a, st) : route_bwd_launch<float, false>(a, st);
}

extern "C" int64_t pp_moe_permute_workspace_ints(int64_t n_slots, int E) {
    if (n_slots < 0 || n_slots > kPermMaxSlots || E < 1 || E > kPermMaxE) return -1;
    return perm_groups(n_slots) * E;
}

extern "C" int pp_moe_permute_ws(const int32_t* expert_of_slot, int64_t n_slots, int E, int32_t* seg_start,
                                 int32_t* row_src, int32_t* pos, int32_t* workspace, int64_t workspace_ints,
                                 pp_stream stream) {
    const int64_t need = pp_moe_permute_workspace_ints(n_slots, E);
    if (need < 0 || !seg_start || (n_slots > 0 && (!expert_of_slot || !row_src || !pos)))
        return fail(PP_ERR_INVALID, "pp_moe_permute_ws: bad arguments (n_slots=%lld E=%d, at most %d experts and %lld slots)",
                    (long long)n_slots, E, kPermMaxE, (long long)kPermMaxSlots);
    if (!workspace || workspace_ints < need)
        return fail(PP_ERR_INVALID, "pp_moe_permute_ws: workspace of %lld ints, needs %lld", (long long)workspace_ints,
                    (long long)need);
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (perm_rounds(n_slots)) {
        case 1: return perm_launch<1>(expert_of_slot, n_slots, E, seg_start, row_src, pos, workspace, st);
        case 2: return perm_launch<2>(expert_of_slot, n_slots, E, seg_start, row_src, pos, workspace, st);
        case 4: return perm_launch<4>(expert_of_slot, n_slots, E, seg_start, row_src, pos, workspace, st);
        default: return perm_launch<8>(expert_of_slot, n_slots, E, seg_start, row_src, pos, workspace, st);
    }
}
