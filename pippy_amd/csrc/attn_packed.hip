// Attention over packed sequences of different lengths (forward, and a deterministic backward in two kernels).
//
// The rows of all sequences lie one after the other, sequence b in rows cu[b] .. cu[b+1]-1.  Inside a sequence
//   S = scale q k^T,  P = softmax(S) (causal: over the keys up to the query),  o = P v,  lse = log sum exp S,
//   dv = P^T do,  dP = do v^T,  dS = P (dP - sum_j P dP),  dq = scale dS k,  dk = scale dS^T q,
// and nothing reaches from one sequence into another: a block of rows is loaded through a buffer resource that
// ends with its sequence, so rows past the end read as zeros whatever the memory behind them holds, and rows
// that belong to no sequence are neither read nor written.
//
// Scores are produced transposed, S^T[key][query], so that a lane holds one query column: softmax statistics
// are per-lane scalars and the probabilities sit in registers as the second product wants its operand.
//
// Which work-group takes which block is a plan built on the device once per batch (pp_attn_packed_plan) and
// shared by all layers and both directions: the blocks of all sequences, the dearest first, so that a launch begins
// with its longest work-groups and fills up with ever shorter ones, however unequal the sequences are.
#include "attn_tile.h"
#include <math.h>

namespace pp {

constexpr int kPlanHeader = 4;   // int32: number of entries of each of the four lists
constexpr int kPlanBins = 2048;  // block indexes from here on count as one length class
constexpr int kPlanThreads = 1024;

// Chunk swizzle of a staged tile: row bits 1, 2, 3 reversed.  Rows start 32 of 64 banks apart.  A ds_read_b128 of one
// chunk of 32 rows is served 16 lanes at a time, rows 0-3, 12-15, 20-27 and the rest: in either set the even rows, and
// the odd ones, get eight different chunks.  A transposing read takes 32 lanes, 4 rows of 4 chunks aligned to 4: rows
// two apart differ in the chunk's bit 2.  (Counted conflicts: SQ_LDS_BANK_CONFLICT 33 % of the active LDS cycles of
// the forward with the swizzle of attn.hip.)
__device__ __forceinline__ int swz_packed(int r) { return ((r & 2) << 1) | ((r & 4) >> 1) | ((r & 8) >> 3); }

struct PackedArgs {
    const uint16_t* q; const uint16_t* k; const uint16_t* v;
    uint16_t* o; float* lse;
    const uint16_t* d_o;
    uint16_t* dq; uint16_t* dk; uint16_t* dv;
    float* delta;
    int64_t sq, sk, sv, so, sdo, sdq, sdk, sdv;  // elements between consecutive rows
    int64_t T;
    int32_t H, G;       // query heads; query heads per key / value head
    const int32_t* plan;
    int32_t cap64, cap128;  // entries that the plan reserves for blocks of 64 and of 128 rows
    float scale;
};

__host__ __device__ inline int64_t plan_blocks64(int64_t T, int64_t n_seq) { return T / 64 + n_seq; }
__host__ __device__ inline int64_t plan_blocks128(int64_t T, int64_t n_seq) { return T / 128 + n_seq; }

// ---- the plan -----------------------------------------------------------------------------------
// Four lists, one work-group each: blocks of 64 and of 128 rows, in the order for a causal mask and in the order
// without one.  Entries {first row of the sequence, its length, block index, 0}, dearest blocks first: under a causal
// mask a block costs as many steps as its index says, without one as its sequence has blocks.  A counting sort over
// that; a wave takes a sequence at a time, its lanes the blocks.  The order inside a class is left to the atomics,
// since it only says which work-group does what.  Bound by latency (two passes over the bounds, a scan, barriers):
// 4.5 us for 4001 rows in 13 sequences as for 16384 in 3; one work-group for all lists took 6.1.
__global__ __launch_bounds__(kPlanThreads) void attn_packed_plan_kernel(const int32_t* __restrict__ cu, int n_seq,
                                                                        int T, int32_t* __restrict__ plan,
                                                                        int cap64, int cap128) {
    __shared__ int cursor[kPlanBins];
    __shared__ int part[kPlanThreads];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    constexpr int kWaves = kPlanThreads / 64;
    const bool wide = blockIdx.x & 1, full = blockIdx.x >> 1;
    const int block = wide ? 128 : 64, cap = wide ? cap128 : cap64;
    int4* entries = reinterpret_cast<int4*>(plan + kPlanHeader) + (full ? cap64 + cap128 : 0) + (wide ? cap64 : 0);
    for (int i = tid; i < kPlanBins; i += kPlanThreads) cursor[i] = 0;
    __syncthreads();
    for (int place = 0; place < 2; ++place) {
        for (int b = wave; b < n_seq; b += kWaves) {
            // bounds that are out of order or out of range make an empty sequence
            const int r0 = cu[b], r1 = cu[b + 1];
            const int len = (r0 >= 0 && r1 > r0 && r1 <= T) ? r1 - r0 : 0;
            const int nb = len / block + (len % block != 0);
            for (int j = lane; j < nb; j += 64) {
                const int cost = full ? nb - 1 : j;
                const int at = atomicAdd(&cursor[cost < kPlanBins - 1 ? cost : kPlanBins - 1], 1);
                if (place && (uint32_t)at < (uint32_t)cap) entries[at] = make_int4(r0, len, j, 0);
            }
        }
        __syncthreads();
        if (place) break;
        // counts -> first places: a class begins behind all dearer ones (two classes per thread)
        const int hi = kPlanBins - 1 - 2 * tid, lo = hi - 1;
        const int n_hi = cursor[hi], n_lo = cursor[lo];
        part[tid] = n_hi + n_lo;
        __syncthreads();
        for (int o = 1; o < kPlanThreads; o <<= 1) {
            const int add = tid >= o ? part[tid - o] : 0;
            __syncthreads();
            part[tid] += add;
            __syncthreads();
        }
        const int begin = part[tid] - n_hi - n_lo;
        cursor[hi] = begin;
        cursor[lo] = begin + n_hi;
        if (tid == kPlanThreads - 1) plan[blockIdx.x] = (uint32_t)part[tid] < (uint32_t)cap ? part[tid] : cap;
        __syncthreads();
    }
}
static_assert(kPlanBins == 2 * kPlanThreads, "the scan takes two classes per thread");

// One block of rows of one sequence, and one head, for a work-group.
struct PackedBlock {
    int64_t row0;  // first row of the sequence
    int len, j;    // its length; index of the block inside it
    int h;
};

// With a multiple of 8 heads every XCD takes its own heads (keys and values of a head in one L2; the heads of a
// group that shares them are neighbours), longest block of all its heads first.  Otherwise the blocks are dealt
// out in order: consecutive work-groups go to different XCDs, and every XCD gets an equal share of each length.
template <bool CAUSAL, bool WIDE>
__device__ __forceinline__ bool packed_block_of(const PackedArgs& a, int heads, PackedBlock* w) {
    const int4* entries = reinterpret_cast<const int4*>(a.plan + kPlanHeader) + (CAUSAL ? 0 : a.cap64 + a.cap128) +
                          (WIDE ? a.cap64 : 0);
    const int n_blocks = a.plan[(CAUSAL ? 0 : 2) + (WIDE ? 1 : 0)];
    const uint32_t bid = blockIdx.x;
    uint32_t t, h;
    if (heads % 8 == 0) {
        const uint32_t g = (uint32_t)heads / 8;
        h = (bid & 7) * g + (bid >> 3) % g;
        t = (bid >> 3) / g;
    } else {
        t = bid / (uint32_t)heads;
        h = bid % (uint32_t)heads;
    }
    const int4 e = entries[t];  // (the grid ends with the list, so this is inside it; one wait for both loads)
    w->row0 = __builtin_amdgcn_readfirstlane(e.x);
    w->len = __builtin_amdgcn_readfirstlane(e.y);
    w->j = __builtin_amdgcn_readfirstlane(e.z);
    w->h = (int)h;
    // a plan that was not made for this call: nothing outside the tensors is touched
    return (t < (uint32_t)n_blocks) & (w->row0 >= 0) & (w->row0 + w->len <= a.T) & (w->j >= 0) &
           ((int64_t)w->j * (WIDE ? 128 : 64) < w->len);
}

// Loader of 64-row blocks of a sequence.  Every block gets a resource of its own that begins at the block (so
// 32-bit offsets suffice however long the sequence is) and ends with the sequence (rows past it read as zeros).
template <int DS>
struct PackedTileLoader {
    const uint16_t* base;
    int64_t stride;
    int len;
    int voff[2];
    __device__ __forceinline__ void init(const uint16_t* first, int64_t stride_, int len_, int wave, int lane) {
        base = first;
        stride = stride_;
        len = len_;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = (i * 4 + wave) * 8 + (lane >> 3);
            voff[i] = row * (int)(stride_ * 2) + (((lane & 7) ^ swz_packed(row)) << 4);
        }
    }
    __device__ __forceinline__ void load(uint16_t* lds, int row0, int wave, int64_t extra = 0) const {
        const int left = len - row0;  // none: a resource of no bytes, everything reads as zeros
        const __amdgpu_buffer_rsrc_t rsrc =
            make_rsrc(base + (int64_t)row0 * stride + extra,
                      left <= 0 ? 0 : (uint64_t)(left < 64 ? left : 64) * (uint64_t)stride * 2);
#pragma unroll
        for (int s = 0; s < DS; ++s)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                load_to_lds_b128(rsrc, lds + s * kTile + (i * 4 + wave) * 512, voff[i] + s * 128, 0);
    }
};

// ---- forward ------------------------------------------------------------------------------------
// A work-group owns 64 query rows of one head and walks the keys in blocks of 64.  Its 4 waves are 2 groups of
// 32 queries x 2 halves of every key block; the two waves of a group merge once, through LDS: a sequence's last
// block takes half as long as with a wave over all its keys, and short sequences fill twice the SIMDs.  Bound by
// the longest work-group's chain of steps (about 0.5 us each: loads, scores, exponentials, the second product).
// 37 rows, 12 heads of 64: 4.5 us; [4001 rows in 13 sequences, 12 heads], no mask: 16.5 us; [4096
// rows in 11 documents, 12 heads], causal: 14.1 us.
template <int D, bool CAUSAL>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void attn_packed_fwd_kernel(const PackedArgs a) {
    constexpr int KS = D / 16, DT = D / 32, DS = D / 64, NS = attn_stages(D);
    constexpr int kOperand = DS * kTile, kStage = 2 * kOperand;
    uint16_t* const lds = attn_lds;

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int grp = wave & 1, half = wave >> 1;
    const int l32 = lane & 31, lh = lane >> 5;
    PackedBlock w;
    if (!packed_block_of<CAUSAL, false>(a, a.H, &w)) return;
    const int q0 = w.j * 64, qw0 = q0 + 32 * grp, qi = qw0 + l32;
    const int hk = w.h / a.G;

    PackedTileLoader<DS> lk, lv;
    lk.init(a.k + w.row0 * a.sk + (int64_t)hk * D, a.sk, w.len, wave, lane);
    lv.init(a.v + w.row0 * a.sv + (int64_t)hk * D, a.sv, w.len, wave, lane);
    const int n_blocks = CAUSAL ? w.j + 1 : (w.len + 63) / 64;
    auto issue = [&](int stage, int j) {
        lk.load(lds + stage * kStage, j * 64, wave);
        lv.load(lds + stage * kStage + kOperand, j * 64, wave);
    };

    // a query past the end computes with the last row and is not stored
    const int qr = qi < w.len ? qi : w.len - 1;
    const uint16_t* qp = a.q + (w.row0 + qr) * a.sq + (int64_t)w.h * D;
    bf16x8_t qf[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = *reinterpret_cast<const bf16x8_t*>(qp + 16 * ks + 8 * lh);
#pragma unroll
    for (int t = 0; t < NS - 1; ++t)
        if (t < n_blocks) issue(t, t);

    f32x16_t oacc[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) oacc[t][e] = 0.f;
    float m_run = -INFINITY, l_run = 0.f;  // l_run: this lane's share of the row sum
    const float c = a.scale * kLog2e;
    const int partner = (lane ^ 32) << 2;

    // this wave's 32 keys of the block from key j * 64 on; MASKED: keys past the last visible one are left out
    auto step = [&](auto masked_c, const uint16_t* Ks, int j) __attribute__((always_inline)) {
        const uint16_t* Vs = Ks + kOperand;
        f32x16_t sacc;
#pragma unroll
        for (int e = 0; e < 16; ++e) sacc[e] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const bf16x8_t kf = read_row_frag<swz_packed>(Ks + (ks / 4) * kTile, 32 * half + l32, 2 * (ks % 4) + lh);
            sacc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[ks], sacc, 0, 0, 0);
        }
        // sacc[v]: key 64 j + 32 half + 8 (v / 4) + 4 lh + v % 4, query qi
        if constexpr (decltype(masked_c)::value) {
            const int lim = (CAUSAL ? qr : w.len - 1) - j * 64 - 32 * half - 4 * lh;
#pragma unroll
            for (int v = 0; v < 16; ++v)
                if (8 * (v >> 2) + (v & 3) > lim) sacc[v] = -INFINITY;
        }
        float mloc = -INFINITY;
#pragma unroll
        for (int v = 0; v < 16; ++v) mloc = fmaxf(mloc, sacc[v]);
        // the reference maximum only keeps the exponentials in range: it moves when a row exceeds it by 2^8
        if (__ballot(mloc * c > m_run * c + 8.0f)) {
            mloc = fmaxf(mloc, __int_as_float(__builtin_amdgcn_ds_bpermute(partner, __float_as_int(mloc))));
            const float m_new = fmaxf(m_run, mloc);
            const float alpha = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m_run - m_new) * c);
            l_run *= alpha;
            m_run = m_new;
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) oacc[t][e] *= alpha;
        }
        const float mc = (m_run == -INFINITY ? 0.f : m_run) * c;
        float psum = 0.f;
#pragma unroll
        for (int v = 0; v < 16; ++v) {
            sacc[v] = __builtin_amdgcn_exp2f(fmaf(sacc[v], c, -mc));
            psum += sacc[v];
        }
        l_run += psum;
#pragma unroll
        for (int gp = 0; gp < 2; ++gp) {
            float pv[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) pv[e] = sacc[8 * gp + e];
            const bf16x8_t pb = pack8(pv);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const bf16x8_t vf = read_col_frag<swz_packed>(Vs + (dt / 2) * kTile, 32 * half + 16 * gp, 32 * (dt % 2), lane);
                oacc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pb, oacc[dt], 0, 0, 0);
            }
        }
    };
    // blocks that every query sees whole, without any masking code; then the diagonal or the end of the sequence
    const int n_whole = CAUSAL ? w.j : w.len / 64;
    int stage = 0, j = 0;
    auto next = [&]() __attribute__((always_inline)) {
        await_block<4 * DS, NS>(j, n_blocks);
        if (j + NS - 1 < n_blocks) issue(stage == 0 ? NS - 1 : stage - 1, j + NS - 1);
        const uint16_t* Ks = lds + stage * kStage;
        stage = stage + 1 == NS ? 0 : stage + 1;
        return Ks;
    };
    for (; j < n_whole; ++j) step(std::false_type{}, next(), j);
    for (; j < n_blocks; ++j) {
        const uint16_t* Ks = next();
        const int kt0 = j * 64 + 32 * half;
        if (kt0 < w.len && (!CAUSAL || kt0 <= qw0 + 31)) step(std::true_type{}, Ks, j);
    }
    l_run += __int_as_float(__builtin_amdgcn_ds_bpermute(partner, __float_as_int(l_run)));

    // merge the two halves in a fixed order: [grp][16 DT + 2 values][64 lanes] floats
    wait_lds();
    __syncthreads();
    float* xs = reinterpret_cast<float*>(lds) + grp * ((16 * DT + 2) * 64) + lane;
    if (half == 1) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e) xs[(16 * dt + e) * 64] = oacc[dt][e];
        xs[16 * DT * 64] = m_run;
        xs[(16 * DT + 1) * 64] = l_run;
    }
    __syncthreads();
    if (half == 1 || qi >= w.len) return;
    const float m1 = xs[16 * DT * 64], l1 = xs[(16 * DT + 1) * 64];
    const float m = fmaxf(m_run, m1);
    const float a0 = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m_run - m) * c);
    const float a1 = m1 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m1 - m) * c);
    const float l = l_run * a0 + l1 * a1, inv_l = 1.0f / l;
    uint16_t* op = a.o + (w.row0 + qi) * a.so + (int64_t)w.h * D;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            float o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                o[e] = (oacc[dt][4 * g + e] * a0 + xs[(16 * dt + 4 * g + e) * 64] * a1) * inv_l;
            const int d = 32 * dt + 8 * g + 4 * lh;
            *reinterpret_cast<uint2*>(op + d) = make_uint2(pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]));
        }
    if (lh == 0) a.lse[(int64_t)w.h * a.T + w.row0 + qi] = m * a.scale + logf(l);
}

// The form for long sequences: a work-group owns 128 query rows, 32 per wave, and every wave walks all keys, in
// blocks of 64: twice the products per staged block and barrier, half the passes over keys and values, and no merge.
// Bound by the matrix cores beside the exponentials: causal [8192 rows, 32 query and 8 key / value heads of 128] 519 us =
// 1060 TFLOP/s of the products it forms (a library product of 8192^3 reaches 1211), 57 % of the cycles in the matrix
// cores, no LDS conflicts; 16384 rows in 3 sequences, 797 to 885 us.
template <int D, bool CAUSAL>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void attn_packed_fwd128_kernel(const PackedArgs a) {
    constexpr int KS = D / 16, DT = D / 32, DS = D / 64, NS = attn_stages(D);
    constexpr int kOperand = DS * kTile, kStage = 2 * kOperand;
    uint16_t* const lds = attn_lds;

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, lh = lane >> 5;
    PackedBlock w;
    if (!packed_block_of<CAUSAL, true>(a, a.H, &w)) return;
    const int q0 = w.j * 128, qw0 = q0 + 32 * wave, qi = qw0 + l32;
    const int hk = w.h / a.G;

    PackedTileLoader<DS> lk, lv;
    lk.init(a.k + w.row0 * a.sk + (int64_t)hk * D, a.sk, w.len, wave, lane);
    lv.init(a.v + w.row0 * a.sv + (int64_t)hk * D, a.sv, w.len, wave, lane);
    const int n_keys = CAUSAL && q0 + 128 < w.len ? q0 + 128 : w.len;
    const int n_blocks = (n_keys + 63) / 64;
    auto issue = [&](int stage, int j) {
        lk.load(lds + stage * kStage, j * 64, wave);
        lv.load(lds + stage * kStage + kOperand, j * 64, wave);
    };

    const int qr = qi < w.len ? qi : w.len - 1;
    const uint16_t* qp = a.q + (w.row0 + qr) * a.sq + (int64_t)w.h * D;
    bf16x8_t qf[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = *reinterpret_cast<const bf16x8_t*>(qp + 16 * ks + 8 * lh);
#pragma unroll
    for (int t = 0; t < NS - 1; ++t)
        if (t < n_blocks) issue(t, t);

    f32x16_t oacc[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) oacc[t][e] = 0.f;
    float m_run = -INFINITY, l_run = 0.f;
    const float c = a.scale * kLog2e;
    const int partner = (lane ^ 32) << 2;
    // keys that some query of this wave sees
    const int seen = CAUSAL && qw0 + 32 < w.len ? qw0 + 32 : w.len;

    // N tiles of 32 keys from key kt0 on, tile rows kr ..; MASKED: keys past the last visible one are left out
    auto step = [&](auto n_c, auto masked_c, const uint16_t* Ks, const uint16_t* Vs, int kr, int kt0)
        __attribute__((always_inline)) {
        constexpr int N = decltype(n_c)::value;
        f32x16_t s[N];
#pragma unroll
        for (int t = 0; t < N; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) s[t][e] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int t = 0; t < N; ++t) {
                const bf16x8_t kf = read_row_frag<swz_packed>(Ks + (ks / 4) * kTile, kr + 32 * t + l32, 2 * (ks % 4) + lh);
                s[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[ks], s[t], 0, 0, 0);
            }
        if constexpr (decltype(masked_c)::value) {
            const int lim = (CAUSAL ? qr : w.len - 1) - kt0 - 4 * lh;
#pragma unroll
            for (int t = 0; t < N; ++t)
#pragma unroll
                for (int v = 0; v < 16; ++v)
                    if (32 * t + 8 * (v >> 2) + (v & 3) > lim) s[t][v] = -INFINITY;
        }
        float mloc = -INFINITY;
#pragma unroll
        for (int t = 0; t < N; ++t)
#pragma unroll
            for (int v = 0; v < 16; ++v) mloc = fmaxf(mloc, s[t][v]);
        if (__ballot(mloc * c > m_run * c + 8.0f)) {
            mloc = fmaxf(mloc, __int_as_float(__builtin_amdgcn_ds_bpermute(partner, __float_as_int(mloc))));
            const float m_new = fmaxf(m_run, mloc);
            const float alpha = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m_run - m_new) * c);
            l_run *= alpha;
            m_run = m_new;
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) oacc[t][e] *= alpha;
        }
        const float mc = (m_run == -INFINITY ? 0.f : m_run) * c;
        float psum = 0.f;
#pragma unroll
        for (int t = 0; t < N; ++t)
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                s[t][v] = __builtin_amdgcn_exp2f(fmaf(s[t][v], c, -mc));
                psum += s[t][v];
            }
        l_run += psum;
#pragma unroll
        for (int t = 0; t < N; ++t)
#pragma unroll
            for (int gp = 0; gp < 2; ++gp) {
                float pv[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) pv[e] = s[t][8 * gp + e];
                const bf16x8_t pb = pack8(pv);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    const bf16x8_t vf = read_col_frag<swz_packed>(Vs + (dt / 2) * kTile, kr + 32 * t + 16 * gp, 32 * (dt % 2), lane);
                    oacc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pb, oacc[dt], 0, 0, 0);
                }
            }
    };
    // Blocks that every query of the work-group sees whole, NS at a time (stages and LDS addresses are constants),
    // without any masking code; then what is left, one tile of 32 keys at a time.
    const int n_whole = (CAUSAL && q0 < w.len ? q0 : w.len) / 64;
    int j = 0;
    for (; j + NS <= n_whole; j += NS)
        static_for<NS>([&](auto stage_c) __attribute__((always_inline)) {
            constexpr int stage = decltype(stage_c)::value;
            await_block<4 * DS, NS>(j + stage, n_blocks);
            if (j + stage + NS - 1 < n_blocks) issue(stage == 0 ? NS - 1 : stage - 1, j + stage + NS - 1);
            step(std::integral_constant<int, 2>{}, std::false_type{}, lds + stage * kStage, lds + stage * kStage + kOperand,
                 0, (j + stage) * 64);
        });
    for (int stage = 0; j < n_blocks; ++j) {
        await_block<4 * DS, NS>(j, n_blocks);
        if (j + NS - 1 < n_blocks) issue(stage == 0 ? NS - 1 : stage - 1, j + NS - 1);
        for (int t = 0; t < 2; ++t)
            if (j * 64 + 32 * t < seen)
                step(std::integral_constant<int, 1>{}, std::true_type{}, lds + stage * kStage,
                     lds + stage * kStage + kOperand, 32 * t, j * 64 + 32 * t);
        stage = stage + 1 == NS ? 0 : stage + 1;
    }
    l_run += __int_as_float(__builtin_amdgcn_ds_bpermute(partner, __float_as_int(l_run)));
    if (qi >= w.len) return;
    const float inv_l = 1.0f / l_run;
    uint16_t* op = a.o + (w.row0 + qi) * a.so + (int64_t)w.h * D;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            float o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = oacc[dt][4 * g + e] * inv_l;
            const int d = 32 * dt + 8 * g + 4 * lh;
            *reinterpret_cast<uint2*>(op + d) = make_uint2(pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]));
        }
    if (lh == 0) a.lse[(int64_t)w.h * a.T + w.row0 + qi] = m_run * a.scale + logf(l_run);
}

// ---- backward: dQ -------------------------------------------------------------------------------
// Fragments of a lane's query row, and delta = rowsum(dO * O) (the lane pair lh = 0, 1 holds the row).
template <int KS>
__device__ __forceinline__ float packed_delta(const uint16_t* qp, const uint16_t* dop, const uint16_t* op, int lh,
                                              bf16x8_t (&qf)[KS], bf16x8_t (&dof)[KS]) {
    float delta = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        qf[ks] = *reinterpret_cast<const bf16x8_t*>(qp + 16 * ks + 8 * lh);
        dof[ks] = *reinterpret_cast<const bf16x8_t*>(dop + 16 * ks + 8 * lh);
        Frag x, y;
        x.v = dof[ks];
        y.u = *reinterpret_cast<const uint4*>(op + 16 * ks + 8 * lh);
        delta += bf16lo(x.u.x) * bf16lo(y.u.x) + bf16hi(x.u.x) * bf16hi(y.u.x) +
                 bf16lo(x.u.y) * bf16lo(y.u.y) + bf16hi(x.u.y) * bf16hi(y.u.y) +
                 bf16lo(x.u.z) * bf16lo(y.u.z) + bf16hi(x.u.z) * bf16hi(y.u.z) +
                 bf16lo(x.u.w) * bf16lo(y.u.w) + bf16hi(x.u.w) * bf16hi(y.u.w);
    }
    return delta + __shfl_xor(delta, 32, 64);
}

// A work-group owns 64 query rows (2 groups of 32 queries x 2 halves of every key block) and hands the dK / dV
// kernel the row sums D = sum_j P dP.  P comes from the stored log-sum-exp, whose rounding, 2^-24 of a number that may be some
// thousands, is one factor on all weights of a row.  From 16 on (a factor of 1 + 2^-20), and with few keys, D is divided by
// sum_j P, so that the row of dS sums to zero all the same.  (Only there: the sum costs up to 2.5 % of the backward.)
//
// dS = P (dP - D), but D is known only behind the loop.  The loop takes delta = rowsum(dO O) of the stored output for it, which
// the rounding of the output keeps from D by r = D - delta, and so leaves a surplus of r P k_j for every key: r times the
// weighted mean of the keys, which dwarfs dQ where weights are nearly even and keys and values have common parts (with
// parts of 16 standard deviations, 2000 keys: an error of 7 times dQ causal, 20 without a mask).  P K is therefore summed beside
// dS K and r P K taken off at the end.  That is a product more per block, of fragments that are there: 4096 rows in 11
// documents, 12 heads of 64: whole backward 40 -> 42 us; 8192 rows in 5 documents, 32 / 8 heads of 128: 548 -> 638 us, where its
// registers also end a form of 128 rows per work-group (with it 1118 us with spills, 671 with one wave per SIMD).
// For head dimension 128 the rows of dO lie in LDS for want of registers (in registers 668 us).
// In a block with one block of keys D is formed before dS.  Bound like the forward's form of 64 rows: 20.4 us for the first of
// these, 305 to 315 for the second (71 % of a library product's rate, 57 % of the cycles in the matrix cores).
template <int D, bool CAUSAL>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void attn_packed_bwd_dq_kernel(const PackedArgs a) {
    constexpr int KS = D / 16, DT = D / 32, DS = D / 64, NS = attn_stages(D);
    constexpr int kOperand = DS * kTile, kStage = 2 * kOperand;
    uint16_t* const lds = attn_lds;

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int grp = wave & 1, half = wave >> 1;
    const int l32 = lane & 31, lh = lane >> 5;
    PackedBlock w;
    if (!packed_block_of<CAUSAL, false>(a, a.H, &w)) return;
    const int q0 = w.j * 64, qw0 = q0 + 32 * grp, qi = qw0 + l32;
    const int hk = w.h / a.G;

    PackedTileLoader<DS> lk, lv;
    lk.init(a.k + w.row0 * a.sk + (int64_t)hk * D, a.sk, w.len, wave, lane);
    lv.init(a.v + w.row0 * a.sv + (int64_t)hk * D, a.sv, w.len, wave, lane);
    const int n_blocks = CAUSAL ? w.j + 1 : (w.len + 63) / 64;
    auto issue = [&](int stage, int j) {
        lk.load(lds + stage * kStage, j * 64, wave);
        lv.load(lds + stage * kStage + kOperand, j * 64, wave);
    };

    const int64_t row = w.row0 + (qi < w.len ? qi : w.len - 1);
    const uint16_t* qp = a.q + row * a.sq + (int64_t)w.h * D;
    const uint16_t* dop = a.d_o + row * a.sdo + (int64_t)w.h * D;
    const uint16_t* op = a.o + row * a.so + (int64_t)w.h * D;
    bf16x8_t qf[KS], dof[KS];
    float delta_q = packed_delta<KS>(qp, dop, op, lh, qf, dof);
    uint16_t* const Ol = lds + NS * kStage;
    if constexpr (D == 128) {
        PackedTileLoader<DS> lo;
        lo.init(a.d_o + w.row0 * a.sdo + (int64_t)w.h * D, a.sdo, w.len, wave, lane);
        lo.load(Ol, q0, wave);
    }
    const float lse_q = a.lse[(int64_t)w.h * a.T + row] * kLog2e;
    float d_sum = 0.f, p_sum = 0.f;
    const bool divide = n_blocks == 1 || __any(fabsf(lse_q) > 16.f * kLog2e);  // (the waves of a group have the same queries)
#pragma unroll
    for (int t = 0; t < NS - 1; ++t)
        if (t < n_blocks) issue(t, t);
    const float c = a.scale * kLog2e;

    f32x16_t dqacc[DT], pkacc[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            dqacc[t][e] = 0.f;
            pkacc[t][e] = 0.f;
        }

    // P and dP of a block; P dP goes into the sum
    auto weights = [&](auto masked_c, const uint16_t* Ks, int j, float (&dsv)[16], f32x16_t& dpacc)
        __attribute__((always_inline)) {
        const uint16_t* Vs = Ks + kOperand;
        f32x16_t sacc;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            sacc[e] = 0.f;
            dpacc[e] = 0.f;
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const bf16x8_t kfr = read_row_frag<swz_packed>(Ks + (ks / 4) * kTile, 32 * half + l32, 2 * (ks % 4) + lh);
            const bf16x8_t vfr = read_row_frag<swz_packed>(Vs + (ks / 4) * kTile, 32 * half + l32, 2 * (ks % 4) + lh);
            sacc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kfr, qf[ks], sacc, 0, 0, 0);
            bf16x8_t of;
            if constexpr (D == 128) of = read_row_frag<swz_packed>(Ol + (ks / 4) * kTile, 32 * grp + l32, 2 * (ks % 4) + lh);
            else of = dof[ks];
            dpacc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vfr, of, dpacc, 0, 0, 0);
        }
#pragma unroll
        for (int v = 0; v < 16; ++v) dsv[v] = __builtin_amdgcn_exp2f(fmaf(sacc[v], c, -lse_q));
        if constexpr (decltype(masked_c)::value) {
            const int lim = (CAUSAL && qi < w.len - 1 ? qi : w.len - 1) - j * 64 - 32 * half - 4 * lh;
#pragma unroll
            for (int v = 0; v < 16; ++v)
                if (8 * (v >> 2) + (v & 3) > lim) dsv[v] = 0.f;
        }
#pragma unroll
        for (int v = 0; v < 16; ++v) d_sum = fmaf(dsv[v], dpacc[v], d_sum);
        if (divide) {
#pragma unroll
            for (int v = 0; v < 16; ++v) p_sum += dsv[v];
        }
    };
    // the row's D from the sums of its lanes and waves; `part`: 256 floats that no load and no other wave uses
    auto row_sum = [&](float* part) __attribute__((always_inline)) {
        d_sum += __shfl_xor(d_sum, 32, 64);
        p_sum += __shfl_xor(p_sum, 32, 64);
        part[wave * 64 + lane] = lh == 0 ? d_sum : p_sum;
        wait_lds();
        __syncthreads();
        const float* row = part + grp * 64 + l32;
        const float d = row[0] + row[128];
        return divide ? d / (row[32] + row[160]) : d;
    };
    auto step = [&](auto masked_c, const uint16_t* Ks, int j) __attribute__((always_inline)) {
        float dsv[16];
        f32x16_t dpacc;
        weights(masked_c, Ks, j, dsv, dpacc);
        const bf16x8_t pb[2] = {pack8(dsv), pack8(dsv + 8)};
#pragma unroll
        for (int v = 0; v < 16; ++v) dsv[v] *= dpacc[v] - delta_q;
#pragma unroll
        for (int gp = 0; gp < 2; ++gp) {
            const bf16x8_t dsb = pack8(dsv + 8 * gp);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const bf16x8_t ktf = read_col_frag<swz_packed>(Ks + (dt / 2) * kTile, 32 * half + 16 * gp, 32 * (dt % 2), lane);
                dqacc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ktf, dsb, dqacc[dt], 0, 0, 0);
                pkacc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ktf, pb[gp], pkacc[dt], 0, 0, 0);
            }
        }
    };
    const int n_whole = CAUSAL ? w.j : w.len / 64;
    int stage = 0, j = 0;
    auto next = [&]() __attribute__((always_inline)) {
        await_block<4 * DS, NS>(j, n_blocks);
        if (j + NS - 1 < n_blocks) issue(stage == 0 ? NS - 1 : stage - 1, j + NS - 1);
        const uint16_t* Ks = lds + stage * kStage;
        stage = stage + 1 == NS ? 0 : stage + 1;
        return Ks;
    };
    if (n_blocks == 1) {
        // Few keys: what the rounding of O leaves in delta weighs most (2 keys: 3.9e-3 of dQ, against 2.3e-3 with the sum),
        // and the sum costs no more than a second look at the one block.
        const uint16_t* Ks = next();
        const bool sees = 32 * half < w.len && (!CAUSAL || 32 * half <= qw0 + 31);
        float pv[16];
        f32x16_t dpv;
        if (sees) weights(std::true_type{}, Ks, 0, pv, dpv);
        delta_q = row_sum(reinterpret_cast<float*>(lds + kStage));  // the second stage, which nothing was loaded into
        d_sum = p_sum = 0.f;
        if (sees) step(std::true_type{}, Ks, 0);
        j = 1;
    }
    for (; j < n_whole; ++j) step(std::false_type{}, next(), j);
    for (; j < n_blocks; ++j) {
        const uint16_t* Ks = next();
        const int kt0 = j * 64 + 32 * half;
        if (kt0 < w.len && (!CAUSAL || kt0 <= qw0 + 31)) step(std::true_type{}, Ks, j);
    }
    // add the sums of the two halves, first the row sums, then [grp][16 DT values][64 lanes] floats
    float* xs = reinterpret_cast<float*>(lds) + grp * (16 * DT * 64) + lane;
    wait_lds();
    __syncthreads();
    const float d_row = row_sum(reinterpret_cast<float*>(lds) + 2 * 16 * DT * 64);
    const float r = d_row - delta_q;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) dqacc[dt][e] = fmaf(-r, pkacc[dt][e], dqacc[dt][e]);
    if (half == 1) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e) xs[(16 * dt + e) * 64] = dqacc[dt][e];
    }
    __syncthreads();
    if (half == 1 || qi >= w.len) return;
    if (lh == 0) a.delta[(int64_t)w.h * a.T + row] = d_row;
    uint16_t* dqp = a.dq + row * a.sdq + (int64_t)w.h * D;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            float s[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] = (dqacc[dt][4 * g + e] + xs[(16 * dt + 4 * g + e) * 64]) * a.scale;
            const int d = 32 * dt + 8 * g + 4 * lh;
            *reinterpret_cast<uint2*>(dqp + d) = make_uint2(pack_bf16(s[0], s[1]), pack_bf16(s[2], s[3]));
        }
}

// ---- backward: dK, dV ---------------------------------------------------------------------------
// A lane holds 16 queries' scores of one key, so log-sum-exp and delta differ from element to element.  They enter the
// products instead, as one more small one: a query's number as three bf16 terms without a remainder (8 bits each) in its
// operand row, against ones.  That is one 4-byte LDS read per lane and statistic where there were four broadcast
// 16-byte ones (a quarter of the kernel's LDS cycles, which bound it beside the matrix cores) and 32 vector
// instructions less: one document of 832 tokens 17.8 -> 14.1 us, [4096 rows, 16 heads of 64] 95 -> 85, [8192, 32 / 8 heads
// of 128] 1093 -> 1026.
typedef short packed_s16x4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ packed_s16x4_t packed_three_parts(float x) {
    const float hi = __uint_as_float(__float_as_uint(x) & 0xffff0000u), rest = x - hi;
    const float mid = __uint_as_float(__float_as_uint(rest) & 0xffff0000u);
    const uint2 w = make_uint2((__float_as_uint(hi) >> 16) | __float_as_uint(mid), __float_as_uint(rest - mid) >> 16);
    return __builtin_bit_cast(packed_s16x4_t, w);
}

// A work-group owns 64 keys of one key / value head and walks the query blocks that see them, one query head of
// the group after the other, so the sums over a group have a fixed order.  4 waves: 2 groups of 32 keys x 2
// halves of every query block.  Head dimension 64.  [4096 rows in 11 documents, 12 heads], causal: 20.5 us, bound by the
// chain of the keys with the most queries behind them (0.85 us a step).
template <bool CAUSAL>
__global__ __launch_bounds__(256, 3) void attn_packed_bwd_dkv_kernel(const PackedArgs a) {
    constexpr int D = 64;
    constexpr int KS = D / 16, DT = D / 32, DS = D / 64, NS = attn_stages(D);
    constexpr int kOperand = DS * kTile;
    constexpr int kStage = 2 * kOperand + 256;  // Q, dO, 64 lse, 64 delta
    uint16_t* const lds = attn_lds;

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int grp = wave & 1, half = wave >> 1;
    const int l32 = lane & 31, lh = lane >> 5;
    PackedBlock w;  // w.h: key / value head
    if (!packed_block_of<CAUSAL, false>(a, a.H / a.G, &w)) return;
    const int nbq = (w.len + 63) / 64;
    // the plan's order is by query work; a key block sees the most queries where a query block sees the fewest
    // keys, so the block index counts from the end here
    const int jk = CAUSAL ? nbq - 1 - w.j : w.j;
    const int kv0 = jk * 64, kvw0 = kv0 + 32 * grp, kvi = kvw0 + l32;
    const int h0 = w.h * a.G;

    PackedTileLoader<DS> lq, ldo;
    lq.init(a.q + w.row0 * a.sq + (int64_t)h0 * D, a.sq, w.len, wave, lane);
    ldo.init(a.d_o + w.row0 * a.sdo + (int64_t)h0 * D, a.sdo, w.len, wave, lane);
    // waves 0 and 2 fetch lse, waves 1 and 3 delta (the same values twice: every wave issues the same number
    // of loads, which keeps the outstanding-load arithmetic uniform)
    const float* stat = ((wave & 1) ? a.delta : a.lse) + (int64_t)h0 * a.T + w.row0;
    const int stat_off = 2 * kOperand + ((wave & 1) ? 128 : 0);

    const int jq0 = CAUSAL ? jk : 0;
    const int nb_head = nbq - jq0, nb = a.G * nb_head;
    int iss_g = 0, iss_b = 0;
    auto issue = [&](int stage) {  // steps are issued in order
        uint16_t* st = lds + stage * kStage;
        const int row0 = (jq0 + iss_b) * 64;
        lq.load(st, row0, wave, (int64_t)iss_g * D);
        ldo.load(st + kOperand, row0, wave, (int64_t)iss_g * D);
        const int left = w.len - row0;
        const __amdgpu_buffer_rsrc_t rs = make_rsrc(stat + (int64_t)iss_g * a.T + row0, (uint64_t)(left < 64 ? left : 64) * 4);
        load_floats_to_lds(rs, reinterpret_cast<float*>(st + stat_off), 0, lane);
        if (++iss_b == nb_head) {
            iss_b = 0;
            ++iss_g;
        }
    };

    const int64_t krow = w.row0 + (kvi < w.len ? kvi : w.len - 1);
    const uint16_t* kp = a.k + krow * a.sk + (int64_t)w.h * D;
    const uint16_t* vp = a.v + krow * a.sv + (int64_t)w.h * D;
    bf16x8_t kf[KS], vf[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        kf[ks] = *reinterpret_cast<const bf16x8_t*>(kp + 16 * ks + 8 * lh);
        vf[ks] = *reinterpret_cast<const bf16x8_t*>(vp + 16 * ks + 8 * lh);
    }
#pragma unroll
    for (int t = 0; t < NS - 1; ++t)
        if (t < nb) issue(t);

    f32x16_t dvacc[DT], dkacc[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            dvacc[t][e] = 0.f;
            dkacc[t][e] = 0.f;
        }
    const float c = a.scale * kLog2e;
    // S - lse / scale and dP - delta come out of the products themselves (see packed_three_parts)
    const float lse_f = lh == 0 ? -1.0f / a.scale : 0.f, delta_f = lh == 0 ? -1.0f : 0.f;
    const packed_s16x4_t ones = {0x3f80, 0x3f80, 0x3f80, 0x3f80};

    // one block of 64 queries from query qb0 on; MASKED: the diagonal block of a causal mask
    auto step = [&](auto masked_c, const uint16_t* Qs, int qb0) __attribute__((always_inline)) {
        const uint16_t* Os = Qs + kOperand;
        const float* lse_s = reinterpret_cast<const float*>(Qs + 2 * kOperand);
        const float* delta_s = lse_s + 64;
        f32x16_t sacc, dpacc;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            sacc[e] = 0.f;
            dpacc[e] = 0.f;
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const bf16x8_t qfr = read_row_frag<swz_packed>(Qs + (ks / 4) * kTile, 32 * half + l32, 2 * (ks % 4) + lh);
            const bf16x8_t ofr = read_row_frag<swz_packed>(Os + (ks / 4) * kTile, 32 * half + l32, 2 * (ks % 4) + lh);
            sacc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(qfr, kf[ks], sacc, 0, 0, 0);
            dpacc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ofr, vf[ks], dpacc, 0, 0, 0);
        }
        sacc = __builtin_amdgcn_mfma_f32_32x32x8bf16_1k(packed_three_parts(lse_s[32 * half + l32] * lse_f), ones, sacc, 0, 0, 0);
        dpacc = __builtin_amdgcn_mfma_f32_32x32x8bf16_1k(packed_three_parts(delta_s[32 * half + l32] * delta_f), ones, dpacc, 0, 0, 0);
        // element v: query qb0 + 32 half + 8 (v / 4) + 4 lh + v % 4, key kvi.  A query past the end has zero rows, a
        // zero log-sum-exp and a zero delta: P = 1 meets dO = 0, dS = 0.
        float pv[16], dsv[16];
#pragma unroll
        for (int v = 0; v < 16; ++v) pv[v] = __builtin_amdgcn_exp2f(sacc[v] * c);
        if constexpr (decltype(masked_c)::value) {
            const int lim = kvi - qb0 - 32 * half - 4 * lh;  // earlier queries do not see this key
#pragma unroll
            for (int v = 0; v < 16; ++v)
                if (8 * (v >> 2) + (v & 3) < lim) pv[v] = 0.f;
        }
#pragma unroll
        for (int v = 0; v < 16; ++v) dsv[v] = pv[v] * dpacc[v];
#pragma unroll
        for (int gp = 0; gp < 2; ++gp) {
            const bf16x8_t pb = pack8(pv + 8 * gp);
            const bf16x8_t dsb = pack8(dsv + 8 * gp);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const bf16x8_t otf = read_col_frag<swz_packed>(Os + (dt / 2) * kTile, 32 * half + 16 * gp, 32 * (dt % 2), lane);
                const bf16x8_t qtf = read_col_frag<swz_packed>(Qs + (dt / 2) * kTile, 32 * half + 16 * gp, 32 * (dt % 2), lane);
                dvacc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(otf, pb, dvacc[dt], 0, 0, 0);
                dkacc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(qtf, dsb, dkacc[dt], 0, 0, 0);
            }
        }
    };
    int stage = 0, j = 0;
    auto next = [&]() __attribute__((always_inline)) {
        await_block<4 * DS + 1, NS>(j, nb);
        if (j + NS - 1 < nb) issue(stage == 0 ? NS - 1 : stage - 1);
        const uint16_t* Qs = lds + stage * kStage;
        stage = stage + 1 == NS ? 0 : stage + 1;
        ++j;
        return Qs;
    };
    // per query head of the group: the diagonal block, then blocks without any masking code
    for (int g = 0; g < a.G; ++g) {
        int b = 0;
        if constexpr (CAUSAL) {
            step(std::true_type{}, next(), jq0 * 64);
            b = 1;
        }
        for (; b < nb_head; ++b) step(std::false_type{}, next(), 0);
    }
    // add the sums of the two halves: [grp][16 DT values][64 lanes] floats, dV then dK
    wait_lds();
    __syncthreads();
    float* xs = reinterpret_cast<float*>(lds) + grp * (16 * DT * 64) + lane;
#pragma unroll
    for (int pass = 0; pass < 2; ++pass) {
        f32x16_t(&acc)[DT] = pass == 0 ? dvacc : dkacc;
        if (half == 1) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int e = 0; e < 16; ++e) xs[(16 * dt + e) * 64] = acc[dt][e];
        }
        __syncthreads();
        if (half == 0 && kvi < w.len) {
            uint16_t* outp = (pass == 0 ? a.dv + krow * a.sdv : a.dk + krow * a.sdk) + (int64_t)w.h * D;
            const float f = pass == 0 ? 1.0f : a.scale;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    float s[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[e] = (acc[dt][4 * g + e] + xs[(16 * dt + 4 * g + e) * 64]) * f;
                    const int d = 32 * dt + 8 * g + 4 * lh;
                    *reinterpret_cast<uint2*>(outp + d) = make_uint2(pack_bf16(s[0], s[1]), pack_bf16(s[2], s[3]));
                }
        }
        __syncthreads();
    }
}

// Head dimension 128: 8 waves per work-group, so that two waves share a SIMD and one's products run beside the
// other's exponentials; to fit the registers of that the value rows stay in LDS.  KB blocks of 64 keys per
// work-group: 2, as 4 groups of 32 keys x 2 parts of a step of 64 queries, or 1, as 2 groups x 4 parts of 128
// queries: twice the work-groups with half the steps each, for launches that would not fill the CUs.  Four
// products per pair of blocks and the exponentials again; 333 to 350 us for causal [8192 rows in 5 documents, 32 query and 8
// key / value heads], 57 % of the cycles in the matrix cores.  Bound by LDS reads beside those; two waves per SIMD is
// what the registers allow.
template <int D, bool CAUSAL, int KB>
__global__ __launch_bounds__(512, 2) void attn_packed_bwd_dkv8_kernel(const PackedArgs a) {
    constexpr int KS = D / 16, DT = D / 32, DS = D / 64, NS = 2;
    constexpr int GROUPS = 2 * KB, PARTS = 8 / GROUPS, QB = PARTS / 2;  // QB: blocks of 64 queries per step
    constexpr int kOperand = DS * kTile;                  // a block of 64 rows
    constexpr int kStats = 2 * QB * kOperand;             // Q blocks, dO blocks, then 64 QB lse, 64 QB delta
    constexpr int kStage = kStats + 256 * QB;
    uint16_t* const lds = attn_lds;
    uint16_t* const Vl = lds + NS * kStage;               // [KB blocks of 64 keys][DS] tiles

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int grp = wave % GROUPS, part = wave / GROUPS;
    const int set = wave >> 2, lwave = wave & 3;          // waves 0-3 load Q, waves 4-7 dO
    const int l32 = lane & 31, lh = lane >> 5;
    PackedBlock w;  // w.h: key / value head
    if (!packed_block_of<CAUSAL, KB == 2>(a, a.H / a.G, &w)) return;
    // the plan's order is by query work; under a causal mask key blocks count from the end (see above)
    const int jk = CAUSAL ? (w.len + 64 * KB - 1) / (64 * KB) - 1 - w.j : w.j;
    const int kv0 = jk * (64 * KB), kvi = kv0 + 32 * grp + l32;
    const int h0 = w.h * a.G;

    PackedTileLoader<DS> lx;
    if (set == 0) lx.init(a.q + w.row0 * a.sq + (int64_t)h0 * D, a.sq, w.len, lwave, lane);
    else lx.init(a.d_o + w.row0 * a.sdo + (int64_t)h0 * D, a.sdo, w.len, lwave, lane);
    const float* stat = (set ? a.delta : a.lse) + (int64_t)h0 * a.T + w.row0;

    constexpr int kStep = 64 * QB;                        // queries per step
    const int u0 = CAUSAL ? kv0 / kStep : 0;              // first step that sees these keys
    const int n_head = (w.len + kStep - 1) / kStep - u0, nb = a.G * n_head;
    int iss_g = 0, iss_b = 0;
    auto issue = [&](int stage) {  // steps are issued in order
        uint16_t* st = lds + stage * kStage;
#pragma unroll
        for (int q = 0; q < QB; ++q) {
            const int row0 = (u0 + iss_b) * kStep + 64 * q;
            // a block past the end loads nothing but zeros, through a resource of no bytes
            lx.load(st + (set * QB + q) * kOperand, row0, lwave, (int64_t)iss_g * D);
            const int left = w.len - row0;
            const __amdgpu_buffer_rsrc_t rs =
                make_rsrc(stat + (int64_t)iss_g * a.T + row0, left <= 0 ? 0 : (uint64_t)(left < 64 ? left : 64) * 4);
            // (every wave of a set the same values: the same number of loads outstanding in each)
            load_floats_to_lds(rs, reinterpret_cast<float*>(st + kStats) + (set * QB + q) * 64, 0, lane);
        }
        if (++iss_b == n_head) {
            iss_b = 0;
            ++iss_g;
        }
    };

    const int64_t krow = w.row0 + (kvi < w.len ? kvi : w.len - 1);
    const uint16_t* kp = a.k + krow * a.sk + (int64_t)w.h * D;
    bf16x8_t kf[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) kf[ks] = *reinterpret_cast<const bf16x8_t*>(kp + 16 * ks + 8 * lh);
    if (set < KB) {  // a set of four waves per block of 64 keys
        PackedTileLoader<DS> lv;
        lv.init(a.v + w.row0 * a.sv + (int64_t)w.h * D, a.sv, w.len, lwave, lane);
        lv.load(Vl + set * kOperand, kv0 + 64 * set, lwave);
    }
    if (nb > 0) issue(0);

    f32x16_t dvacc[DT], dkacc[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            dvacc[t][e] = 0.f;
            dkacc[t][e] = 0.f;
        }
    const float c = a.scale * kLog2e;
    // S - lse / scale and dP - delta come out of the products themselves (see packed_three_parts)
    const float lse_f = lh == 0 ? -1.0f / a.scale : 0.f, delta_f = lh == 0 ? -1.0f : 0.f;
    const packed_s16x4_t ones = {0x3f80, 0x3f80, 0x3f80, 0x3f80};
    const uint16_t* Vs = Vl + (grp >> 1) * kOperand;
    const int vrow = 32 * (grp & 1) + l32;
    const int qblk = part >> 1, half = part & 1;          // this wave's 32 queries of a step

    auto step = [&](auto masked_c, const uint16_t* st, int qb0) __attribute__((always_inline)) {
        const uint16_t* Qs = st + qblk * kOperand;
        const uint16_t* Os = st + (QB + qblk) * kOperand;
        const float* lse_s = reinterpret_cast<const float*>(st + kStats) + 64 * qblk + 32 * half;
        const float* delta_s = lse_s + 64 * QB;
        f32x16_t sacc, dpacc;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            sacc[e] = 0.f;
            dpacc[e] = 0.f;
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const bf16x8_t qfr = read_row_frag<swz_packed>(Qs + (ks / 4) * kTile, 32 * half + l32, 2 * (ks % 4) + lh);
            sacc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(qfr, kf[ks], sacc, 0, 0, 0);
        }
        sacc = __builtin_amdgcn_mfma_f32_32x32x8bf16_1k(packed_three_parts(lse_s[l32] * lse_f), ones, sacc, 0, 0, 0);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const bf16x8_t ofr = read_row_frag<swz_packed>(Os + (ks / 4) * kTile, 32 * half + l32, 2 * (ks % 4) + lh);
            const bf16x8_t vfr = read_row_frag<swz_packed>(Vs + (ks / 4) * kTile, vrow, 2 * (ks % 4) + lh);
            dpacc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ofr, vfr, dpacc, 0, 0, 0);
        }
        dpacc = __builtin_amdgcn_mfma_f32_32x32x8bf16_1k(packed_three_parts(delta_s[l32] * delta_f), ones, dpacc, 0, 0, 0);
        float pv[16], dsv[16];
#pragma unroll
        for (int v = 0; v < 16; ++v) pv[v] = __builtin_amdgcn_exp2f(sacc[v] * c);
        if constexpr (decltype(masked_c)::value) {
            const int lim = kvi - qb0 - 32 * part - 4 * lh;  // earlier queries do not see this key
#pragma unroll
            for (int v = 0; v < 16; ++v)
                if (8 * (v >> 2) + (v & 3) < lim) pv[v] = 0.f;
        }
#pragma unroll
        for (int v = 0; v < 16; ++v) dsv[v] = pv[v] * dpacc[v];
#pragma unroll
        for (int gp = 0; gp < 2; ++gp) {
            const bf16x8_t pb = pack8(pv + 8 * gp);
            const bf16x8_t dsb = pack8(dsv + 8 * gp);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const bf16x8_t otf = read_col_frag<swz_packed>(Os + (dt / 2) * kTile, 32 * half + 16 * gp, 32 * (dt % 2), lane);
                const bf16x8_t qtf = read_col_frag<swz_packed>(Qs + (dt / 2) * kTile, 32 * half + 16 * gp, 32 * (dt % 2), lane);
                dvacc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(otf, pb, dvacc[dt], 0, 0, 0);
                dkacc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(qtf, dsb, dkacc[dt], 0, 0, 0);
            }
        }
    };
    int stage = 0, j = 0;
    auto next = [&]() __attribute__((always_inline)) {
        await_block<QB * (2 * DS + 1), NS>(j, nb);
        if (j + 1 < nb) issue(stage ^ 1);
        const uint16_t* st = lds + stage * kStage;
        stage ^= 1;
        ++j;
        return st;
    };
    // per query head of the group: the steps that the diagonal crosses, then steps without any masking code
    constexpr int kDiag = CAUSAL ? KB / QB > 1 ? KB / QB : 1 : 0;
    for (int g = 0; g < a.G; ++g) {
        int b = 0;
        for (; b < kDiag && b < n_head; ++b) step(std::true_type{}, next(), (u0 + b) * kStep);
        for (; b < n_head; ++b) step(std::false_type{}, next(), 0);
    }
    // add the sums of the parts in a fixed order: [part - 1][grp][16 DT values][64 lanes] floats, dV then dK
    wait_lds();
    __syncthreads();
    float* xs = reinterpret_cast<float*>(lds) + grp * (16 * DT * 64) + lane;
    constexpr int kPart = GROUPS * 16 * DT * 64;
    static_assert((PARTS - 1) * kPart * 4 <= NS * kStage * 2, "the exchange fits the stages");
#pragma unroll
    for (int pass = 0; pass < 2; ++pass) {
        f32x16_t(&acc)[DT] = pass == 0 ? dvacc : dkacc;
        if (part != 0) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int e = 0; e < 16; ++e) xs[(part - 1) * kPart + (16 * dt + e) * 64] = acc[dt][e];
        }
        __syncthreads();
        if (part == 0 && kvi < w.len) {
            uint16_t* outp = (pass == 0 ? a.dv + krow * a.sdv : a.dk + krow * a.sdk) + (int64_t)w.h * D;
            const float f = pass == 0 ? 1.0f : a.scale;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    float s[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[e] = acc[dt][4 * g + e];
#pragma unroll
                        for (int q = 0; q < PARTS - 1; ++q) s[e] += xs[q * kPart + (16 * dt + 4 * g + e) * 64];
                        s[e] *= f;
                    }
                    const int d = 32 * dt + 8 * g + 4 * lh;
                    *reinterpret_cast<uint2*>(outp + d) = make_uint2(pack_bf16(s[0], s[1]), pack_bf16(s[2], s[3]));
                }
        }
        __syncthreads();
    }
}

static constexpr size_t dkv8_lds_bytes(int D, int kb) {
    return (size_t)2 * ((2 / kb) * (2 * (D / 64) * kTile * 2 + 512)) + (size_t)kb * (D / 64) * kTile * 2;
}
static_assert(dkv8_lds_bytes(128, 1) <= 160 * 1024 && dkv8_lds_bytes(128, 2) <= 160 * 1024, "a work-group's LDS");

// ---- entry points -------------------------------------------------------------------------------
static int packed_check(const char* who, const pp_attn_packed_desc* d, bool bwd) {
    if (!d) return fail(PP_ERR_INVALID, "%s: null descriptor", who);
    if (pp_attn_packed_plan_ints(d->n_seq, d->T) < 0 || d->H <= 0 || d->H > (1 << 17) || d->Hkv <= 0 || d->H % d->Hkv)
        return fail(PP_ERR_INVALID, "%s: bad shape (T=%lld n_seq=%lld H=%lld Hkv=%lld)", who, (long long)d->T,
                    (long long)d->n_seq, (long long)d->H, (long long)d->Hkv);
    if (d->D != 64 && d->D != 128)
        return fail(PP_ERR_UNSUPPORTED, "%s: head_dim %lld (64 and 128 are built)", who, (long long)d->D);
    // (log-sum-exp / scale is formed in fp32)
    if (!(d->scale >= 0x1p-64f) || !(d->scale <= 0x1p64f))
        return fail(PP_ERR_INVALID, "%s: scale must be positive and finite, between 2^-64 and 2^64", who);
    const struct { const void* p; int64_t stride, width; const char* name; bool need; } rows[] = {
        {d->q, d->stride_q, d->H * d->D, "q", true},     {d->k, d->stride_k, d->Hkv * d->D, "k", true},
        {d->v, d->stride_v, d->Hkv * d->D, "v", true},   {d->o, d->stride_o, d->H * d->D, "o", true},
        {d->d_o, d->stride_do, d->H * d->D, "d_o", bwd}, {d->dq, d->stride_dq, d->H * d->D, "dq", bwd},
        {d->dk, d->stride_dk, d->Hkv * d->D, "dk", bwd}, {d->dv, d->stride_dv, d->Hkv * d->D, "dv", bwd}};
    if (d->T == 0) return PP_OK;  // (empty tensors have no address)
    for (const auto& r : rows) {
        if (!r.need) continue;
        if (!r.p || !aligned(r.p, 16)) return fail(PP_ERR_INVALID, "%s: %s must be a 16-byte aligned pointer", who, r.name);
        // 64 rows of a block are addressed with 32-bit byte offsets
        if (r.stride % 8 || r.stride < r.width || r.stride > (1 << 23))
            return fail(PP_ERR_INVALID, "%s: row stride %lld of %s must be a multiple of 8 in [%lld, %d]", who,
                        (long long)r.stride, r.name, (long long)r.width, 1 << 23);
    }
    if (!d->lse || !d->plan || !aligned(d->plan, 16) || (bwd && !d->delta))
        return fail(PP_ERR_INVALID, "%s: null pointer, or a plan that is not 16-byte aligned", who);
    if (plan_blocks64(d->T, d->n_seq) * d->H > 0x7fffff00ll) return fail(PP_ERR_UNSUPPORTED, "%s: grid too large", who);
    return PP_OK;
}

static PackedArgs packed_args(const pp_attn_packed_desc* d) {
    PackedArgs a;
    a.q = (const uint16_t*)d->q; a.k = (const uint16_t*)d->k; a.v = (const uint16_t*)d->v;
    a.o = (uint16_t*)d->o; a.lse = d->lse;
    a.d_o = (const uint16_t*)d->d_o;
    a.dq = (uint16_t*)d->dq; a.dk = (uint16_t*)d->dk; a.dv = (uint16_t*)d->dv;
    a.delta = d->delta;
    a.sq = d->stride_q; a.sk = d->stride_k; a.sv = d->stride_v; a.so = d->stride_o;
    a.sdo = d->stride_do; a.sdq = d->stride_dq; a.sdk = d->stride_dk; a.sdv = d->stride_dv;
    a.T = d->T;
    a.H = (int32_t)d->H;
    a.G = (int32_t)(d->H / d->Hkv);
    a.plan = d->plan;
    a.cap64 = (int32_t)plan_blocks64(d->T, d->n_seq);
    a.cap128 = (int32_t)plan_blocks128(d->T, d->n_seq);
    a.scale = d->scale;
    return a;
}

// Dynamic LDS of the forward and dQ kernels: the stages (the exchange of the epilogue is smaller).
static size_t packed_lds_bytes(int D) {
    return (size_t)attn_stages(D) * 2 * (D / 64) * kTile * 2;
}
static_assert(3 * 2 * kTile * 2 >= 2 * (16 * 2 + 2) * 64 * 4 && 2 * 2 * 2 * kTile * 2 >= 2 * (16 * 4 + 2) * 64 * 4,
              "the exchange of two halves fits the stages");

template <auto kernel>
static int packed_launch(const char* name, int threads, int64_t grid, size_t lds, hipStream_t st, const PackedArgs& a) {
    // one attribute call per kernel (the kernel is a template argument, so is the static) and process
    static const hipError_t attr_rc =
        hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (attr_rc != hipSuccess)
        return fail(PP_ERR_LAUNCH, "%s: cannot reserve %zu bytes of LDS: %s", name, lds, hipGetErrorString(attr_rc));
    hipLaunchKernelGGL(kernel, dim3((uint32_t)grid), dim3(threads), lds, st, a);
    return check_launch(name);
}

// The forward's form of 128 rows (for dK / dV 128 keys, below) where the launch has at least as many blocks of 128 as the
// CUs hold work-groups at once (3 of head dimension 64, 2 of 128; the sequences' last, partly filled blocks are left
// out of the count).  With fewer, half as many work-groups leave CUs idle and the last one takes twice as long.  Forward,
// us, 64 rows | 128 rows:
//   D = 64:  [16 heads] T = 2048: 23.7 | 27.6, 4096: 50.6 | 57.4; [12 heads] T = 8192: 150 | 129; [16] T = 16384 in 16
//            sequences: 89.6 | 74.4, in 256: 42.8 | 39.1
//   D = 128: [32 heads] T = 1024: 20.7 | 24.3, 2048: 50.6 | 49.7, 4096: 169 | 141, 16384 in 3 sequences: 1070 | 870
static bool packed_wide(const pp_attn_packed_desc* d, int64_t heads) {
    return d->T / 128 * heads >= (d->D == 64 ? 3 : 2) * 256;
}

template <int D, bool CAUSAL>
static int packed_fwd(const pp_attn_packed_desc* d, hipStream_t st) {
    const PackedArgs a = packed_args(d);
    const size_t lds = packed_lds_bytes(D);
    if (packed_wide(d, d->H))
        return packed_launch<attn_packed_fwd128_kernel<D, CAUSAL>>("attn_packed_fwd128_kernel", 256,
                                                                   plan_blocks128(d->T, d->n_seq) * d->H, lds, st, a);
    return packed_launch<attn_packed_fwd_kernel<D, CAUSAL>>("attn_packed_fwd_kernel", 256,
                                                            plan_blocks64(d->T, d->n_seq) * d->H, lds, st, a);
}

template <int D, bool CAUSAL>
static int packed_bwd(const pp_attn_packed_desc* d, hipStream_t st) {
    const PackedArgs a = packed_args(d);
    constexpr int DS = D / 64;
    const int64_t blocks64 = plan_blocks64(d->T, d->n_seq), blocks128 = plan_blocks128(d->T, d->n_seq);
    // the dQ kernel goes first: it leaves the row sums that the dK / dV kernel reads
    const size_t lds = packed_lds_bytes(D);
    if constexpr (D == 64) {
        const int rc = packed_launch<attn_packed_bwd_dq_kernel<D, CAUSAL>>("attn_packed_bwd_dq_kernel", 256,
                                                                           blocks64 * d->H, lds, st, a);
        if (rc) return rc;
        return packed_launch<attn_packed_bwd_dkv_kernel<CAUSAL>>("attn_packed_bwd_dkv_kernel", 256, blocks64 * d->Hkv,
                                                                 attn_stages(D) * (2 * kTile * 2 + 512), st, a);
    } else {
        const int rc = packed_launch<attn_packed_bwd_dq_kernel<D, CAUSAL>>("attn_packed_bwd_dq_kernel", 256, blocks64 * d->H,
                                                                           lds + DS * kTile * 2, st, a);
        if (rc) return rc;
        // Whole backward, causal, us, 64 | 128 keys per work-group: [32 query, 8 key / value heads] T = 2048: 202 | 272, 4096: 555 |
        // 668, 8192: 2096 | 2022, in 5 sequences: 625 | 644, 16384 in 16: 963 | 885; [32, 32] T = 1024: 64 | 66, 2048: 176 | 160
        if (packed_wide(d, d->Hkv))
            return packed_launch<attn_packed_bwd_dkv8_kernel<D, CAUSAL, 2>>("attn_packed_bwd_dkv8_kernel", 512,
                                                                            blocks128 * d->Hkv, dkv8_lds_bytes(D, 2), st, a);
        return packed_launch<attn_packed_bwd_dkv8_kernel<D, CAUSAL, 1>>("attn_packed_bwd_dkv8_kernel", 512,
                                                                        blocks64 * d->Hkv, dkv8_lds_bytes(D, 1), st, a);
    }
}

}  // namespace pp

using namespace pp;

extern "C" int64_t pp_attn_packed_plan_ints(int64_t n_seq, int64_t T) {
    if (n_seq < 0 || T < 0 || n_seq > 0x7fffffc0ll || T > 0x7fffffc0ll) return -1;
    const int64_t entries = 2 * (plan_blocks64(T, n_seq) + plan_blocks128(T, n_seq));
    return entries > 0x7fffffffll ? -1 : kPlanHeader + 4 * entries;
}

extern "C" int pp_attn_packed_plan(const int32_t* cu_seqlens, int64_t n_seq, int64_t T, int32_t* plan, pp_stream stream) {
    if (pp_attn_packed_plan_ints(n_seq, T) < 0)
        return fail(PP_ERR_INVALID, "pp_attn_packed_plan: bad shape (n_seq=%lld T=%lld)", (long long)n_seq, (long long)T);
    if (!plan || !aligned(plan, 16) || (n_seq > 0 && !cu_seqlens))
        return fail(PP_ERR_INVALID, "pp_attn_packed_plan: null pointer, or a plan that is not 16-byte aligned");
    hipLaunchKernelGGL(attn_packed_plan_kernel, dim3(4), dim3(kPlanThreads), 0, static_cast<hipStream_t>(stream),
                       cu_seqlens, (int)n_seq, (int)T, plan, (int)plan_blocks64(T, n_seq), (int)plan_blocks128(T, n_seq));
    return check_launch("attn_packed_plan_kernel");
}

extern "C" int pp_attn_packed_fwd(const pp_attn_packed_desc* d, pp_stream stream) {
    const int rc = packed_check("pp_attn_packed_fwd", d, false);
    if (rc) return rc;
    if (d->T == 0 || d->n_seq == 0) return PP_OK;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (d->D == 64) return d->causal ? packed_fwd<64, true>(d, st) : packed_fwd<64, false>(d, st);
    return d->causal ? packed_fwd<128, true>(d, st) : packed_fwd<128, false>(d, st);
}

extern "C" int pp_attn_packed_bwd(const pp_attn_packed_desc* d, pp_stream stream) {
    const int rc = packed_check("pp_attn_packed_bwd", d, true);
    if (rc) return rc;
    if (d->T == 0 || d->n_seq == 0) return PP_OK;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (d->D == 64) return d->causal ? packed_bwd<64, true>(d, st) : packed_bwd<64, false>(d, st);
    return d->causal ? packed_bwd<128, true>(d, st) : packed_bwd<128, false>(d, st);
}
