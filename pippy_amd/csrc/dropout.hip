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

template <typename ET>
__device__ __forceinline__ float dropout_load(const void* p, int64_t i) {
    if constexpr (sizeof(ET) == 2) return bf16_to_f32(static_cast<const uint16_t*>(p)[i]);
    else return static_cast<const float*>(p)[i];
}

// A dropped element contributes a zero whatever it holds (an infinity or NaN too).
template <typename ET>
__global__ __launch_bounds__(256) void dropout_kernel(const DropoutArgs a) {
    const uint64_t seed = a.rng[0], offset = a.rng[1];
    const int64_t per_row = (a.C + 7) / 8, n = a.rows * per_row;
    for (int64_t g = (int64_t)blockIdx.x * 256 + threadIdx.x; g < n; g += (int64_t)gridDim.x * 256) {
        float f[8];
        dropout_factors(a, seed, offset, (uint32_t)g, f);
        const int64_t r = g / per_row, c0 = (g % per_row) * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (c0 + e >= a.C) break;
            float v = a.resid ? dropout_load<ET>(a.resid, r * a.ld_r + c0 + e) : 0.f;
            if (f[e] != 0.f) v = fmaf(dropout_load<ET>(a.x, r * a.ld_x + c0 + e), f[e], v);
            if constexpr (sizeof(ET) == 2) static_cast<uint16_t*>(a.y)[r * a.ld_y + c0 + e] = f32_to_bf16(v);
            else static_cast<float*>(a.y)[r * a.ld_y + c0 + e] = v;
        }
    }
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
    const int64_t blocks = (rows * ((C + 7) / 8) + 255) / 256;
    const dim3 grid((unsigned)(blocks < 65536 ? blocks : 65536));
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == PP_BF16) hipLaunchKernelGGL(dropout_kernel<uint16_t>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(dropout_kernel<float>, grid, dim3(256), 0, st, a);
    return check_launch("dropout_kernel");
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
