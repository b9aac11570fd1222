// Dropout with an optional residual, from a counter-based generator; the mask is never stored.
//   y = resid + m x / (1 - p'),   dx = m dy / (1 - p')
// m comes from Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011) on
// the counter {element / 8, offset (64 bits), site} under the key {seed (64 bits)}: one call makes the 16-bit draws
// of 8 consecutive elements, and an element stays when its draw is at least the border round(65536 p).  16 bits
// per element quantise the rate to p' = border / 65536 (the scale uses p', so the expectation is exact); 32 bits
// would double the integer products.  Backward and forward of a site make the same mask from the same
// {seed, offset}, which live in device memory: a captured graph or a launch list replays with whatever values
// they hold then.
#include "common.h"

namespace pp {

__device__ __forceinline__ uint4 philox_10(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}

struct DropoutArgs {
    const void* x; const void* resid; void* y;
    const uint64_t* rng;  // {seed, offset}
    int64_t rows, C, ld_x, ld_r, ld_y;
    uint32_t site, border;
    float scale;
};

// The 8 factors (0 or scale) of a group of consecutive elements.
__device__ __forceinline__ void dropout_factors(const DropoutArgs& a, uint64_t seed, uint64_t offset, uint32_t group,
                                                float (&f)[8]) {
    const uint4 r = philox_10(group, (uint32_t)offset, (uint32_t)(offset >> 32), a.site, (uint32_t)seed,
                              (uint32_t)(seed >> 32));
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = (w[i] & 0xffffu) >= a.border ? a.scale : 0.f;
        f[2 * i + 1] = (w[i] >> 16) >= a.border ? a.scale : 0.f;
    }
}

// A dropped element contributes a zero whatever it holds (an infinity or NaN too).  In bf16 the work is one 16-byte
// access per tensor and group; FLAT: one row, whose elements are addressed without a division.
template <typename ET>
struct DropoutVec;
template <>
struct DropoutVec<uint16_t> {
    uint4 w;
    __device__ __forceinline__ void load(const void* p, int64_t i) {
        w = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
    }
    __device__ __forceinline__ void unpack(float (&v)[8]) const {
        v[0] = bf16lo(w.x); v[1] = bf16hi(w.x); v[2] = bf16lo(w.y); v[3] = bf16hi(w.y);
        v[4] = bf16lo(w.z); v[5] = bf16hi(w.z); v[6] = bf16lo(w.w); v[7] = bf16hi(w.w);
    }
    static __device__ __forceinline__ void store(void* p, int64_t i, const float (&v)[8]) {
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) =
            make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
    }
    static __device__ __forceinline__ float load1(const void* p, int64_t i) {
        return bf16_to_f32(static_cast<const uint16_t*>(p)[i]);
    }
    static __device__ __forceinline__ void store1(void* p, int64_t i, float v) {
        static_cast<uint16_t*>(p)[i] = f32_to_bf16(v);
    }
};
template <>
struct DropoutVec<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const void* p, int64_t i) {
        const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
        a = q[0];
        b = q[1];
    }
    __device__ __forceinline__ void unpack(float (&v)[8]) const {
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
    static __device__ __forceinline__ void store(void* p, int64_t i, const float (&v)[8]) {
        float4* q = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
        q[0] = make_float4(v[0], v[1], v[2], v[3]);
        q[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
    static __device__ __forceinline__ float load1(const void* p, int64_t i) { return static_cast<const float*>(p)[i]; }
    static __device__ __forceinline__ void store1(void* p, int64_t i, float v) { static_cast<float*>(p)[i] = v; }
};

// Bound by HBM: bf16 [16384, 4096] with a residual 69 to 75 us (5.4 to 5.8 TB/s over 403 MB), without one 45 us (5.9 TB/s);
// the generator's 20 wide products per 8 elements hide behind that.  [1021, 768]: 3 us, latency.
constexpr int kDropoutGroups = 2;  // groups of 8 elements per lane: their loads are all in flight at once

template <typename ET, bool FLAT, bool RESID>
__global__ __launch_bounds__(256) void dropout_kernel(const DropoutArgs a) {
    const uint64_t seed = a.rng[0], offset = a.rng[1];
    const uint32_t per_row = (uint32_t)((a.C + 7) / 8);
    const uint64_t n = (uint64_t)a.rows * (uint64_t)((a.C + 7) / 8), n_whole = FLAT ? (uint64_t)a.C / 8 : n;
    const uint64_t g0 = (uint64_t)blockIdx.x * (256 * kDropoutGroups) + threadIdx.x;
    DropoutVec<ET> x[kDropoutGroups], r[kDropoutGroups];
    uint32_t row[kDropoutGroups], col[kDropoutGroups];
#pragma unroll
    for (int q = 0; q < kDropoutGroups; ++q) {
        const uint64_t g = g0 + q * 256;
        row[q] = 0;
        col[q] = 0;
        if (g >= n_whole) continue;
        if constexpr (!FLAT) {
            row[q] = (uint32_t)g / per_row;  // fewer than 2^32 groups
            col[q] = (uint32_t)g % per_row;
        }
        x[q].load(a.x, FLAT ? (int64_t)g * 8 : row[q] * a.ld_x + (int64_t)col[q] * 8);
        if constexpr (RESID) r[q].load(a.resid, FLAT ? (int64_t)g * 8 : row[q] * a.ld_r + (int64_t)col[q] * 8);
    }
#pragma unroll
    for (int q = 0; q < kDropoutGroups; ++q) {
        const uint64_t g = g0 + q * 256;
        if (g >= n) continue;
        float f[8];
        dropout_factors(a, seed, offset, (uint32_t)g, f);
        if (g < n_whole) {
            float v[8], t[8], y[8];
            x[q].unpack(v);
            if constexpr (RESID) r[q].unpack(t);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float kept = f[e] != 0.f ? v[e] : 0.f;
                y[e] = RESID ? fmaf(kept, f[e], t[e]) : kept * f[e];
            }
            DropoutVec<ET>::store(a.y, FLAT ? (int64_t)g * 8 : row[q] * a.ld_y + (int64_t)col[q] * 8, y);
        } else {  // the last elements of a flat tensor whose length is no multiple of 8
            for (int e = 0; e < 8 && (int64_t)g * 8 + e < a.C; ++e) {
                const int64_t i = (int64_t)g * 8 + e;
                float v = RESID ? DropoutVec<ET>::load1(a.resid, i) : 0.f;
                if (f[e] != 0.f) v = fmaf(DropoutVec<ET>::load1(a.x, i), f[e], v);
                DropoutVec<ET>::store1(a.y, i, v);
            }
        }
    }
}

template <typename ET>
static int dropout_launch(const DropoutArgs& a, hipStream_t st) {
    const int64_t groups = a.rows * ((a.C + 7) / 8), per_block = 256 * kDropoutGroups;
    const dim3 grid((unsigned)((groups + per_block - 1) / per_block));
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, a);
        return check_launch("dropout_kernel");
    };
    if (a.rows == 1) return a.resid ? go(dropout_kernel<ET, true, true>) : go(dropout_kernel<ET, true, false>);
    return a.resid ? go(dropout_kernel<ET, false, true>) : go(dropout_kernel<ET, false, false>);
}

__global__ void rng_advance_kernel(uint64_t* rng, uint64_t step) { rng[1] += step; }

static int dropout_run(const char* who, const void* x, int64_t ld_x, const void* resid, int64_t ld_r, void* y,
                       int64_t ld_y, int64_t rows, int64_t C, int dtype, float p, const uint64_t* rng, uint32_t site,
                       pp_stream stream) {
    if (dtype != PP_BF16 && dtype != PP_F32) return fail(PP_ERR_INVALID, "%s: unknown dtype %d", who, dtype);
    if (!(p >= 0.f) || !(p <= 1.f)) return fail(PP_ERR_INVALID, "%s: p must lie in [0, 1]", who);
    if (rows < 0 || C < 0) return fail(PP_ERR_INVALID, "%s: bad shape", who);
    if (rows == 0 || C == 0) return PP_OK;
    if (!x || !y || !rng || !aligned(rng, 8) || !aligned(x, 16) || !aligned(y, 16) || !aligned(resid, 16))
        return fail(PP_ERR_INVALID, "%s: null pointer, or one that is not aligned (16 bytes; rng 8)", who);
    if (rows > 1 && (C % 8 || ld_x % 8 || ld_y % 8 || (resid && ld_r % 8) || ld_x < C || ld_y < C || (resid && ld_r < C)))
        return fail(PP_ERR_INVALID, "%s: several rows need widths and leading dimensions that are multiples of 8 (C=%lld)",
                    who, (long long)C);
    if (C > (1ll << 35) || rows > (1ll << 35) / ((C + 7) / 8 * 8))
        return fail(PP_ERR_UNSUPPORTED, "%s: more than 2^35 elements", who);
    DropoutArgs a;
    a.x = x; a.resid = resid; a.y = y; a.rng = rng;
    a.rows = rows; a.C = C; a.ld_x = ld_x; a.ld_r = ld_r; a.ld_y = ld_y;
    a.site = site;
    // p = 1 drops everything; a smaller p never rounds up to that
    const uint32_t border = (uint32_t)(p * 65536.0f + 0.5f);
    a.border = p >= 1.f ? 65536u : (border > 65535u ? 65535u : border);
    a.scale = p >= 1.f ? 0.f : 65536.0f / (float)(65536u - a.border);
    hipStream_t st = static_cast<hipStream_t>(stream);
    return dtype == PP_BF16 ? dropout_launch<uint16_t>(a, st) : dropout_launch<float>(a, st);
}

}  // namespace pp

using namespace pp;

extern "C" int pp_dropout_add(const void* x, int64_t ld_x, const void* resid, int64_t ld_resid, void* y, int64_t ld_y,
                              int64_t rows, int64_t C, int dtype, float p, const uint64_t* rng, uint32_t site,
                              pp_stream stream) {
    return dropout_run("pp_dropout_add", x, ld_x, resid, ld_resid, y, ld_y, rows, C, dtype, p, rng, site, stream);
}

extern "C" int pp_dropout_bwd(const void* dy, int64_t ld_dy, void* dx, int64_t ld_dx, int64_t rows, int64_t C, int dtype,
                              float p, const uint64_t* rng, uint32_t site, pp_stream stream) {
    return dropout_run("pp_dropout_bwd", dy, ld_dy, nullptr, 0, dx, ld_dx, rows, C, dtype, p, rng, site, stream);
}

extern "C" int pp_rng_advance(uint64_t* rng, uint64_t step, pp_stream stream) {
    if (!rng || !aligned(rng, 8)) return fail(PP_ERR_INVALID, "pp_rng_advance: null or misaligned pointer");
    hipLaunchKernelGGL(rng_advance_kernel, dim3(1), dim3(1), 0, static_cast<hipStream_t>(stream), rng, step);
    return check_launch("rng_advance_kernel");
}
