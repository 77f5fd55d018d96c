// Which expert and which rows a workgroup works on, found on the device from the experts' row
// offsets, so that the host never has to know them (no copy, no synchronisation, capturable).
//
// The rows 0 .. N - 1 are cut into E + 2 segments: rows before offsets[0], the E experts, rows
// from offsets[E] on.  Each segment is cut into tiles of `tile` rows; a launch has
// ragged_tiles(N, E, tile) of them at most.
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>

namespace forge {

// full tiles, and at most one partial tile per segment that has rows
static inline int64_t ragged_tiles(int64_t N, int64_t E, int64_t tile) {
    const int64_t segments = E + 2 < N ? E + 2 : N;
    return N / tile + segments;
}

struct RaggedTile {
    int expert;      // -1: rows of no expert
    int row0, rows;  // first row of the tile, rows in it (1 .. tile)
    int p;           // which tile of the other operand
};

__device__ __forceinline__ int clamp_offset(const int32_t* offsets, int i, int lo, int N) {
    int v = offsets[i];
    v = v < lo ? lo : v;
    return v > N ? N : v;
}

// A segment's first row, its end and the number of its tiles; the number of a segment of `light` rows or fewer
// (one tile) is in the upper half
__device__ __forceinline__ uint64_t segment_tiles(const int32_t* offsets, int s, int E, int N, int tile, int light, int& a, int& b) {
    a = b = 0;
    if (s >= E + 2) return 0;
    a = s == 0 ? 0 : clamp_offset(offsets, s - 1, 0, N);
    b = s == E + 1 ? N : clamp_offset(offsets, s, a, N);
    const unsigned rows = (unsigned)(b - a);
    if (rows > 0 && rows <= (unsigned)light) return (uint64_t)1 << 32;
    return (rows + (unsigned)tile - 1) / (unsigned)tile;
}

// Called by all 512 threads of a workgroup.  Every tile of rows meets p_tiles tiles of the other operand;
// which(T, L) names, from the numbers of products of ordinary segments and of light ones, the one this
// workgroup takes (0 .. T - 1, then T .. T + L - 1; anything else: none, and false is returned).  A segment's
// products follow one another, with up to 8 of its tiles by all of p_tiles side by side: an XCD's 32 workgroups
// then read the segment's weights once, and 12 panels or fewer in all.  `slot` is LDS of the caller's.
// Offsets outside [0, N] or descending are clamped: no tile reaches out of [0, N).
struct FindSlot {
    uint64_t waves[8];
    int out[4], chunk[8];
};
template <typename F>
__device__ __forceinline__ bool find_tile(const int32_t* __restrict__ offsets, int E, int N, int tile, int light, int p_tiles, F which,
                                          RaggedTile& out, FindSlot& slot) {
    const int id = threadIdx.x, lane = id & 63, wave = id >> 6;
    int a, b;
    const uint64_t first_run = segment_tiles(offsets, id, E, N, tile, light, a, b);
    uint64_t total = first_run;
    for (int s = id + 512; s < E + 2; s += 512) {
        int x, y;
        total += segment_tiles(offsets, s, E, N, tile, light, x, y);
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) total += __shfl_xor(total, d);
    if (lane == 0) slot.waves[wave] = total;
    if (id == 0) slot.out[2] = 0;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) total += slot.waves[w];
    const int full = (int)(uint32_t)total * p_tiles, few = (int)(total >> 32) * p_tiles;
    int i = which(full, few);
    if (i < 0 || i >= full + few) return false;                   // the same in every thread
    const bool is_light = i >= full;
    if (is_light) i -= full;
    const int t = i / p_tiles;                                    // in the segment that holds this tile
    int before = 0;
    uint64_t both = first_run;
    for (int s0 = 0;; s0 += 512) {
        if (s0) both = segment_tiles(offsets, s0 + id, E, N, tile, light, a, b);
        const int mine = is_light ? (int)(both >> 32) : (int)(uint32_t)both;
        int upto = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int v = __shfl_up(upto, d);
            if (lane >= d) upto += v;
        }
        if (lane == 63) slot.chunk[wave] = upto;
        __syncthreads();
        int first = before + upto - mine;
#pragma unroll
        for (int w = 0; w < 8; ++w) {
            if (w < wave) first += slot.chunk[w];
            before += slot.chunk[w];
        }
        if (mine > 0 && t >= first && t < first + mine) {
            const int local = i - first * p_tiles, groups = (mine + 7) / 8, wide = (mine + groups - 1) / groups;
            const int group = local / (wide * p_tiles), in_group = local - group * wide * p_tiles;
            const int here = mine - group * wide < wide ? mine - group * wide : wide;
            const int r0 = a + (group * wide + in_group % here) * tile;
            slot.out[0] = s0 + id - 1 < E ? s0 + id - 1 : -1;
            slot.out[1] = r0;
            slot.out[2] = b - r0 < tile ? b - r0 : tile;
            slot.out[3] = in_group / here;
        }
        __syncthreads();
        if (before > t || s0 + 512 >= E + 2) break;
    }
    // the same for every lane: in scalar registers from here on
    out.expert = __builtin_amdgcn_readfirstlane(slot.out[0]);
    out.row0 = __builtin_amdgcn_readfirstlane(slot.out[1]);
    out.rows = __builtin_amdgcn_readfirstlane(slot.out[2]);
    out.p = __builtin_amdgcn_readfirstlane(slot.out[3]);
    return out.rows > 0;
}

}  // namespace forge
