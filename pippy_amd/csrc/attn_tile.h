// Tile helpers of the attention kernels (equal sequences: attn.hip; packed sequences: attn_packed.hip): 64 x 64 bf16
// tiles in LDS exactly as they lie in memory, direct-to-LDS loads, and the fragment reads of
// v_mfma_f32_32x32x16_bf16 along either index of a tile.
#pragma once
#include "tile.h"

namespace pp {

union Frag {
    uint4 u;
    bf16x8_t v;
};
__device__ __forceinline__ bf16x8_t pack8(const float* p) {
    Frag f;
    f.u = make_uint4(pack_bf16(p[0], p[1]), pack_bf16(p[2], p[3]), pack_bf16(p[4], p[5]),
                     pack_bf16(p[6], p[7]));
    return f.v;
}

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kTile = 64 * 64;  // elements of one staged tile
// LDS stages: 3 x 16 KiB for head dimension 64 (three work-groups per CU), 2 x 32 KiB for 128
constexpr int attn_stages(int D) { return D == 64 ? 3 : 2; }

// Chunk swizzle of a staged tile.  Rows r and r+1 start 32 banks apart; the first term spreads 16
// consecutive rows read at one chunk index (ds_read_b128 fragments), the second separates rows r
// and r+2, which a transposing read touches together.
__device__ __forceinline__ int swz_attn(int r) { return ((r ^ (r >> 3)) & 7) ^ ((r & 2) << 1); }

// Direct-to-LDS loader of 64-row blocks out of a [rows][stride] operand: DS tiles of 64 columns
// (128 B per row and tile), tile s at lds + s * kTile.
// ASM: the loads go out as inline assembly (see tile.h), which lets tiles stay in flight across LDS reads.
// Measured on the three kernels it changed nothing (forward 1.92 against 1.95 ms, backward 5.12 against
// 5.29 ms per GPT-2-small step, within the scatter between machines): a work-group's chain of dependent
// block steps, not its loads, sets the pace.  The kernels stay on the builtin form.
template <int DS, bool ASM = false>
struct AttnTileLoader {
    typename std::conditional<ASM, LdsDmaRsrc, __amdgpu_buffer_rsrc_t>::type rsrc;
    int voff[2];
    int row_bytes;
    __device__ __forceinline__ void init(const uint16_t* base, int64_t stride, int64_t rows, int wave, int lane) {
        if constexpr (ASM) rsrc = make_lds_dma_rsrc(base, (uint64_t)rows * (uint64_t)stride * 2);
        else rsrc = make_rsrc(base, (uint64_t)rows * (uint64_t)stride * 2);
        row_bytes = (int)(stride * 2);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = (i * 4 + wave) * 8 + (lane >> 3);
            voff[i] = row * row_bytes + (((lane & 7) ^ swz_attn(row)) << 4);
        }
    }
    // `extra_bytes` shifts the columns (another head of the same rows)
    __device__ __forceinline__ void load(uint16_t* lds, int64_t row0, int wave, int extra_bytes = 0) const {
#pragma unroll
        for (int s = 0; s < DS; ++s)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                load_to_lds_b128(rsrc, lds + s * kTile + (i * 4 + wave) * 512, voff[i] + s * 128,
                                 (int)row0 * row_bytes + extra_bytes);
    }
};

// 64 consecutive floats into LDS with one wave instruction.
__device__ __forceinline__ void load_floats_to_lds(__amdgpu_buffer_rsrc_t rsrc, float* lds, int64_t first, int lane) {
#if defined(__HIP_DEVICE_COMPILE__)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void_ptr_t)lds, 4, lane * 4, (int)first * 4, 0, 0);
#endif
}

// Fragment with k along d: row `row` of the tile, 16-byte chunk `chunk`.
template <int (*SWZ)(int) = swz_attn>
__device__ __forceinline__ bf16x8_t read_row_frag(const uint16_t* tile, int row, int chunk) {
    return *reinterpret_cast<const bf16x8_t*>(tile + row * 64 + ((chunk ^ SWZ(row)) << 3));
}

// Fragment with k along the tile's rows, for 32 columns d0 .. d0+31 and the 16 rows r0 .. r0+15.
// The k slots of lane group g = lane / 32 are rows r0 + 4g .. + 3 and r0 + 8 + 4g .. + 3: the order
// in which a lane of a 32x32 MFMA result holds 8 of its 16 values, so that probabilities computed
// in registers can be the other operand without a shuffle.  Inside each block of 16 lanes, lane
// 4j + i fetches columns 4i .. 4i+3 of row j, and the hardware hands lane m the 4 rows of column m.
template <int (*SWZ)(int) = swz_attn>
__device__ __forceinline__ bf16x8_t read_col_frag(const uint16_t* tile, int r0, int d0, int lane) {
#if defined(__HIP_DEVICE_COMPILE__)
    const int g = lane >> 5, mb = (lane >> 4) & 1, j = (lane & 15) >> 2, i = lane & 3;
    const int d = d0 + 16 * mb + 4 * i;
    const int r_lo = r0 + 4 * g + j, r_hi = r_lo + 8;
    const uint16_t* p_lo = tile + r_lo * 64 + (((d >> 3) ^ SWZ(r_lo)) << 3) + (d & 7);
    const uint16_t* p_hi = tile + r_hi * 64 + (((d >> 3) ^ SWZ(r_hi)) << 3) + (d & 7);
    const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr_t)p_lo);
    const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr_t)p_hi);
    const s16x8_t v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(bf16x8_t, v);
#else
    return bf16x8_t{};
#endif
}

// Pipeline step shared by the three kernels: block j of `nb` has landed for every wave, and the
// stage that block j-1 occupied is free.  LPT loads per block per wave; with NS stages, NS - 2
// younger blocks may stay in flight.
template <int LPT, int NS>
__device__ __forceinline__ void await_block(int64_t j, int64_t nb) {
    static_assert(NS == 2 || NS == 3, "two or three stages");
    if (NS == 3 && j + 1 < nb) wait_vmcnt<(NS == 3 ? LPT : 0)>(); else wait_vmcnt<0>();
    wait_lds();
    __builtin_amdgcn_s_barrier();
}

extern __shared__ __attribute__((aligned(16))) uint16_t attn_lds[];

}  // namespace pp
