// Which expert and which rows a workgroup works on, found on the device from the experts' row
// offsets, so that the host never has to know them (no copy, no synchronisation, capturable).
//
// The rows 0 .. N - 1 are cut into E + 2 segments: rows before offsets[0], the E experts, rows
// from offsets[E] on.  Each segment is cut into tiles of `tile` rows; tile t of the launch is the
// t-th of that list.  A launch has ragged_tiles(N, E, tile) of them at most.
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
};

__device__ __forceinline__ int clamp_offset(const int32_t* offsets, int i, int lo, int N) {
    int v = offsets[i];
    v = v < lo ? lo : v;
    return v > N ? N : v;
}

// A segment's first row and the number of its tiles
__device__ __forceinline__ int segment_tiles(const int32_t* offsets, int s, int E, int N, int tile, int& a, int& b) {
    a = b = 0;
    if (s >= E + 2) return 0;
    a = s == 0 ? 0 : clamp_offset(offsets, s - 1, 0, N);
    b = s == E + 1 ? N : clamp_offset(offsets, s, a, N);
    return (int)(((unsigned)(b - a) + (unsigned)tile - 1u) / (unsigned)tile);
}

// Called by every thread of a workgroup: which(T) names, from the number T of tiles there are, the one
// this workgroup takes (negative or >= T: none; then false).  `slot` is LDS of the caller's.
// Offsets outside [0, N] or descending are clamped: no tile reaches out of [0, N).
template <typename F>
__device__ __forceinline__ bool find_tile(const int32_t* __restrict__ offsets, int E, int N, int tile, F which,
                                          RaggedTile& out, int* slot) {
    if (threadIdx.x < 64) {
        const int lane = threadIdx.x;
        int a, b, total = 0;
        const int first_run = segment_tiles(offsets, lane, E, N, tile, a, b);
        total = first_run;
        for (int s = lane + 64; s < E + 2; s += 64) {
            int x, y;
            total += segment_tiles(offsets, s, E, N, tile, x, y);
        }
#pragma unroll
        for (int d = 32; d; d >>= 1) total += __shfl_xor(total, d);
        const int t = which(total);
        if (lane == 0) slot[2] = 0;
        if (t >= 0 && t < total) {
            int before = 0, mine = first_run;
            for (int s0 = 0;; s0 += 64) {
                if (s0) mine = segment_tiles(offsets, s0 + lane, E, N, tile, a, b);
                int upto = mine;
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) {
                    const int v = __shfl_up(upto, d);
                    if (lane >= d) upto += v;
                }
                const int first = before + upto - mine;
                if (mine > 0 && t >= first && t < first + mine) {
                    const int r0 = a + (t - first) * tile;
                    slot[0] = s0 + lane - 1 < E ? s0 + lane - 1 : -1;
                    slot[1] = r0;
                    slot[2] = b - r0 < tile ? b - r0 : tile;
                }
                before += __shfl(upto, 63);
                if (before > t || s0 + 64 >= E + 2) break;
            }
        }
    }
    __syncthreads();
    // the same for every lane: in scalar registers from here on
    out.expert = __builtin_amdgcn_readfirstlane(slot[0]);
    out.row0 = __builtin_amdgcn_readfirstlane(slot[1]);
    out.rows = __builtin_amdgcn_readfirstlane(slot[2]);
    return out.rows > 0;
}

}  // namespace forge
