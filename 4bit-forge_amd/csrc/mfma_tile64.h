// 256 x 256 tiles of a bf16 product for the 32x32x16 matrix instruction: how a 64-deep stage of
// either operand lies in LDS, how it gets there, and how a wavefront reads its fragments.
//
// A workgroup is 8 wavefronts, 2 along P (the operand that runs along the accumulator's registers)
// by 4 along Q (the one that runs across the lanes): 128 x 64 outputs each, 8 matrix instructions
// per 6 fragments.  Per stage that is 192 KB of LDS reads for 2048 clocks of matrix work at 128
// bytes a clock, so the matrix pipe and not the LDS is the limit; 64 x 64 per wavefront (16
// wavefronts) would need 256 KB and sit exactly on it.
//
// Stages go from memory to LDS without touching registers (buffer_load ... lds, 16 bytes a lane):
// the next stage's loads are issued before the current stage is multiplied.  A lane whose element
// lies outside the matrix gets an offset beyond the descriptor's range, for which the hardware
// writes zeros.
//
// The lanes of one such load write 1 KiB of consecutive LDS, so the layout that keeps the reads free of
// bank conflicts is made by choosing which 16 bytes each lane fetches:
//   K_INNER (the inner dimension is contiguous in memory): 256 rows of 128 bytes; 16-byte piece c of
//     row r lies at piece c ^ (r / 2 % 8), so 16 consecutive rows of one piece cover all 64 banks.
//   K_OUTER (the inner dimension is the row): 64 rows of 512 bytes, read transposed by
//     ds_read_b64_tr_b16 (16 lanes fetch 4 rows x 16 columns, lane i receives column i); piece c of
//     row k lies at c ^ 4 (k % 4), so that the four rows of one read are in different banks.
#pragma once
#include "act.h"

namespace forge {

constexpr int kTile = 256;        // outputs of a workgroup in either direction
constexpr int kStage = 64;        // inner dimension of a stage
constexpr int kStageBytes = kTile * kStage * 2;
constexpr uint32_t kOutside = 0x80000000u;   // an offset beyond every descriptor's range

typedef __attribute__((address_space(3))) char lds_char;
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4;

__device__ __forceinline__ __amdgpu_buffer_rsrc_t descriptor(const void* p, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)bytes, 0x00020000);
}
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t d, char* lds, uint32_t offset) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(d, (__attribute__((address_space(3))) void*)lds, 16, (int)offset, 0, 0, 0);
}
// everything this wavefront has on its way to LDS has arrived
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(0x0F70); }   // vmcnt(0)

// ---- K_INNER: rows `row0 ..` of a matrix with pitch ld, inner dimension `inner`
struct InnerLoader {
    uint32_t off[4];     // byte offset of this lane's 16 bytes of the four loads of its wavefront
    uint32_t piece[4];   // and their place in the stage (columns)
    // `rows` valid rows (others read as zero); row_of(r): which row of the descriptor tile row r is
    template <typename F>
    __device__ __forceinline__ void init(int wave, int lane, int64_t ld, int rows, F row_of) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int r = (wave * 4 + j) * 8 + lane / 8;
            const int c = (lane & 7) ^ ((r >> 1) & 7);
            const int m = row_of(r);
            piece[j] = c * 8;
            off[j] = m < rows ? (uint32_t)(m * ld * 2) + c * 16 : kOutside;
        }
    }
    __device__ __forceinline__ void stage(__amdgpu_buffer_rsrc_t d, char* lds, int wave, int k0, int inner) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t o = k0 + (int)piece[j] < inner ? off[j] + (uint32_t)k0 * 2 : kOutside;
            load_to_lds(d, lds + (wave * 4 + j) * 1024, o);
        }
    }
};
// ---- K_OUTER: columns `col0 ..` of a matrix whose rows are the inner dimension.  The descriptor is
// made per stage (base at the stage's first row), so row offsets never pass 32 bits.
struct OuterLoader {
    uint32_t off[4];
    __device__ __forceinline__ void init(int wave, int lane, int64_t ld, int cols) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k = (wave * 4 + j) * 2 + lane / 32;
            const int c = (lane & 31) ^ ((k & 3) << 2);
            off[j] = c * 8 < cols ? (uint32_t)(k * ld * 2) + c * 16 : kOutside;
        }
    }
    // base: first row of the stage at the tile's first column; rows left in the matrix from there
    __device__ __forceinline__ void stage(const uint16_t* base, int64_t ld, int left, int cols, char* lds, int wave) const {
        const int rows = left < kStage ? left : kStage;
        const int width = cols < kTile ? cols : kTile;
        const __amdgpu_buffer_rsrc_t d = descriptor(base, (uint32_t)(((rows - 1) * ld + width) * 2));
#pragma unroll
        for (int j = 0; j < 4; ++j) load_to_lds(d, lds + (wave * 4 + j) * 1024, off[j]);
    }
};

// ---- fragments: 32 rows (tile t of the operand) x 16 of the inner dimension (step s of the stage)
struct InnerFragment {
    uint32_t at[4];
    __device__ __forceinline__ void init(int lane, int tile0) {
        const int r = lane & 31;
#pragma unroll
        for (int s = 0; s < 4; ++s)
            at[s] = (tile0 * 32 + r) * 128 + (((2 * s + (lane >> 5)) ^ ((r >> 1) & 7)) * 16);
    }
    __device__ __forceinline__ bf16x8_t read(const char* lds, int t, int s) const {
        return *reinterpret_cast<const bf16x8_t*>(lds + at[s] + t * 4096);
    }
};
template <int TILES>
struct OuterFragment {
    uint32_t at[TILES];
    __device__ __forceinline__ void init(int lane, int tile0) {
        const int g = lane >> 4, i = lane & 15;
        const int k = 8 * (g >> 1) + (i >> 2);                    // k % 4 = i / 4
        const int col = 16 * (g & 1) + 4 * (i & 3);
#pragma unroll
        for (int t = 0; t < TILES; ++t)
            at[t] = k * 512 + ((((col >> 3) + (tile0 + t) * 4) ^ ((i >> 2) << 2)) * 16) + (col & 7) * 2;
    }
    __device__ __forceinline__ bf16x8_t read(const char* lds, int t, int s) const {
        const char* p = lds + at[t] + s * 8192;
        const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
        const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 2048));
        typedef short s16x8 __attribute__((ext_vector_type(8)));
        const s16x8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        return __builtin_bit_cast(bf16x8_t, v);
    }
};

// One stage: 4 steps of 16, 4 x 2 matrix instructions each.
template <typename FP, typename FQ>
__device__ __forceinline__ void multiply_stage(const char* P, const char* Q, const FP& fp, const FQ& fq,
                                               f32x16_t (&acc)[4][2]) {
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        bf16x8_t p[4], q[2];
#pragma unroll
        for (int t = 0; t < 4; ++t) p[t] = fp.read(P, t, s);
#pragma unroll
        for (int t = 0; t < 2; ++t) q[t] = fq.read(Q, t, s);
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int n = 0; n < 2; ++n)
                acc[t][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(p[t], q[n], acc[t][n], 0, 0, 0);
    }
}

// Workgroup b of a launch runs on XCD b % 8 (each has its own L2): gives every XCD a run of
// consecutive tiles, so that tiles that share an operand share an L2.
__device__ __forceinline__ int xcd_tile(int b, int blocks) {
    const int q = blocks / 8, r = blocks % 8, x = b % 8;
    return x * q + (x < r ? x : r) + b / 8;
}

}  // namespace forge
