// Gated feed-forward rows of routed experts and their gradients.
//
//   forward    g = X_e Wg[e]^T,  u = X_e Wu[e]^T,  h = act(g) * u
//   backward   dg = dh * u * act'(g),  du = dh * act(g)
//              dX_e = dg Wg[e] + du Wu[e],  dWg[e] = dg^T X_e,  dWu[e] = du^T X_e
//
// Three products over one ragged batch.  All run on the bf16 matrix instruction with f32 sums.
#include "act.h"
#include "common.h"
#include "mfma_tile.h"
#include "ragged.h"
#include <type_traits>

namespace {
using forge::act_f32;
using forge::act_grad_f32;
using forge::bf16x8_t;
using forge::f32_to_bf16_bits;
using forge::f32x16_t;
using forge::f32x4_t;
using forge::find_tile;
using forge::pack_bf16;
using forge::RaggedTile;

struct GatedArgs {
    const uint16_t* x;       // rows [N, H], pitch ldx
    const int32_t* offsets;  // [E + 1]
    const uint16_t* wg;      // [E, I, H], pitch ldw, stride ws
    const uint16_t* wu;
    int64_t ldx, ldw, ws;
    int N, E, H, I, act;
    uint16_t* h;             // forward: [N, I]
    float* g;                // forward: may be null
    float* u;
    const uint16_t* dg;      // backward: [N, I]
    const uint16_t* du;
    uint16_t* dx;            // [N, H]
    uint16_t* dwg;           // [E, I, H], dense
    uint16_t* dwu;
};

enum { FORWARD = 0, DROWS = 1, DWEIGHTS = 2 };
constexpr int kLightRows = 128;   // an expert with that many rows or fewer takes half a full tile's matrix work at most

// ---------------------------------------------------------------- many rows
// 256 x 256 outputs per workgroup (mfma_tile.h).  P runs along the registers of the accumulator, i.e. along
// the output's contiguous dimension, Q across the lanes:
//   FORWARD   P = weight rows, Q = rows of X,              inner dimension H
//   DROWS     P = columns of X, Q = rows of X,             inner I, twice
//   DWEIGHTS  P = columns of X, Q = rows of dW,            inner the expert's rows
// with
//   FORWARD   P = 128 features: tile rows 128 w .. + 63 are Wg's rows 64 w .., the next 64 Wu's, so
//             that wavefront w of P holds g and u of the same features in the same lanes and the
//             activation and the product need no exchange
//   DROWS     P and Q of the gate, then of the up projection, into the same sums
// The inner dimension's tail and rows or columns outside are zeros that the loads themselves write.
// Measured: FORWARD 32768 rows of one expert, 7168 x 1024, 722 us, 1334 TFLOP/s (the card's power limit, 1.6 GHz); 16384
// rows of 16 experts by popularity, 7168 x 2048, 860 us; 32768 rows of 128 experts, 2048 x 768, 290 us, 1.35 GB from
// beyond L2.  DROWS 8168 rows of 16 experts, 7168 x 2048, 495 us.  DWEIGHTS 8192 rows of one expert 365 us.
template <int MODE>
__global__ __launch_bounds__(512) void gated_tile_kernel(GatedArgs a, int p_tiles, int q_tiles) {
    using namespace forge;
    __shared__ __attribute__((aligned(1024))) char P0[kStageBytes], P1[kStageBytes], P2[kStageBytes], Q0[kStageBytes], Q1[kStageBytes];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // wavefronts i and i + 4 share a SIMD; they get different quarters of Q, so that a tile with few rows
    // keeps one wavefront busy on every SIMD instead of two on some
    const int wp = wave >> 2, wq = (wave & 3) ^ (wp << 1);

    RaggedTile r;
    int q0 = 0, inner = 0, which = 0, pt;
    if constexpr (MODE == DWEIGHTS) {
        // experts differ in rows, so every XCD takes an eighth of every expert's tiles
        const int tiles = p_tiles * q_tiles, per = (tiles + 7) / 8;
        const int i = blockIdx.x / 8, t = (blockIdx.x % 8) * per + i % per;
        if (t >= tiles) return;
        r.expert = (i / per) % a.E;
        which = (i / per) / a.E;
        pt = t % p_tiles;
        q0 = (t / p_tiles) * kTile;
        r.row0 = clamp_offset(a.offsets, r.expert, 0, a.N);
        r.rows = clamp_offset(a.offsets, r.expert + 1, r.row0, a.N) - r.row0;
        inner = r.rows;
    } else {
        if (!find_tile(a.offsets, a.E, a.N, kTile, kLightRows, p_tiles, [&](int full, int light) {
                int t;
                return xcd_tile(blockIdx.x, full, light, t) ? t : full + t;
            }, r, *reinterpret_cast<FindSlot*>(P2))) return;
        __syncthreads();                                          // P2 is read
        pt = r.p;
        inner = r.expert < 0 ? 0 : MODE == FORWARD ? a.H : a.I;
    }
    const int p0 = pt * (MODE == FORWARD ? kTile / 2 : kTile);
    const int per_phase = (inner + kStage - 1) / kStage;
    // nothing to sum (rows of no expert, an expert without rows): one stage of zeros
    const int stages = max(MODE == DROWS ? 2 * per_phase : per_phase, 1);
    const int64_t we = (int64_t)(r.expert < 0 ? 0 : r.expert) * a.ws;
    const bool light = MODE != DWEIGHTS && r.rows <= 64;

    // loaders
    InnerLoader<4> lp_in, lq_in;
    OuterLoader<> lp_out, lq_out;
    __amdgpu_buffer_rsrc_t dp, dq;
    if constexpr (MODE == FORWARD) {
        const bool up = (wave & 3) >= 2;                       // this wavefront loads rows of Wu
        const int rows = a.I - p0 < kTile / 2 ? a.I - p0 : kTile / 2;
        lp_in.init(lane, a.ldw, (wave >> 2) * 64 + (wave & 1) * 32);
        dp = descriptor((up ? a.wu : a.wg) + we + (int64_t)p0 * a.ldw, (uint32_t)(((rows - 1) * a.ldw + a.H) * 2));
        lq_in.init(lane, a.ldx, wave * 32);
        dq = descriptor(a.x + (int64_t)r.row0 * a.ldx, (uint32_t)(((r.rows - 1) * a.ldx + a.H) * 2));
    } else if constexpr (MODE == DROWS) {
        lp_out.init(wave, lane, a.ldw, a.H - p0);
        lq_in.init(lane, a.I, wave * 32);
    } else {
        lp_out.init(wave, lane, a.ldx, a.H - p0);
        lq_out.init(wave, lane, a.I, a.I - q0);
    }
    auto load_p = [&](int s, char* P) {
        if constexpr (MODE == FORWARD) {
            lp_in.stage(dp, P, wave, a.ldw, s * kStage, inner);
        } else if constexpr (MODE == DROWS) {
            const bool up = s >= per_phase;
            const int k0 = (up ? s - per_phase : s) * kStage;
            lp_out.stage((up ? a.wu : a.wg) + we + (int64_t)k0 * a.ldw + p0, a.ldw, inner - k0, a.H - p0, P, wave);
        } else {
            const int64_t k0 = (int64_t)r.row0 + s * kStage;
            lp_out.stage(a.x + k0 * a.ldx + p0, a.ldx, r.rows - s * kStage, a.H - p0, P, wave);
        }
    };
    auto load_q_by = [&](const auto& loader, int s, char* Q) {
        if constexpr (MODE == FORWARD) {
            loader.stage(dq, Q, wave, a.ldx, s * kStage, inner);
        } else if constexpr (MODE == DROWS) {
            const bool up = s >= per_phase;
            const int k0 = (up ? s - per_phase : s) * kStage;
            const __amdgpu_buffer_rsrc_t d = descriptor((up ? a.du : a.dg) + (int64_t)r.row0 * a.I, (uint32_t)(r.rows * a.I * 2));
            loader.stage(d, Q, wave, a.I, k0, inner);
        } else {
            const int64_t k0 = (int64_t)r.row0 + s * kStage;
            loader.stage((which ? a.du : a.dg) + k0 * a.I + q0, a.I, r.rows - s * kStage, a.I - q0, Q, wave);
        }
    };
    auto load_q = [&](int s, char* Q) {
        if constexpr (MODE == DWEIGHTS) load_q_by(lq_out, s, Q); else load_q_by(lq_in, s, Q);
    };
    // Registers 4 j .. 4 j + 3 of a tile: rows 8 j + 4 (lane / 32) .. + 3 of P, column lane & 31 of Q, i.e.
    // 8 bytes of 32 rows of the output at a time.  Every wavefront's part goes through 16 KB of LDS of its own,
    // [row of Q][K pieces of 16 bytes], with the pieces of a row in an order that keeps the banks apart, and
    // leaves in whole rows of it.
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    lds_char* mine = (wave < 4 ? wave < 2 ? (lds_char*)P0 : (lds_char*)P1 : wave < 6 ? (lds_char*)P2 : (lds_char*)Q0) + (wave & 1) * 16384;
    auto place = [](auto pieces, int row, int piece) {
        constexpr int K = decltype(pieces)::value, kShift = K == 16 ? 0 : K == 8 ? 1 : 2;
        return row * (K * 16) + ((piece ^ ((row >> kShift) & (K - 1))) * 16);
    };
    // 32 columns (block) x 32 rows (from row0 on) of the wavefront's part of the output; FORWARD: from g and u
    auto put = [&](auto pieces, int row0, int block, const f32x16_t& x, const f32x16_t& y) {
        // an opaque copy: addresses made from it are not formed before the inner loop, where they would
        // cost registers
        int lane_e = lane;
        asm volatile("" : "+v"(lane_e));
        float h[16];
        if constexpr (MODE == FORWARD) {
            act_times(a.act, x, y, h);
        } else {
#pragma unroll
            for (int v = 0; v < 16; ++v) h[v] = x[v];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            *(__attribute__((address_space(3))) u32x2*)(mine + place(pieces, row0 + (lane_e & 31), block * 4 + j) + (lane_e >> 5) * 8) =
                u32x2{pack_bf16(h[4 * j], h[4 * j + 1]), pack_bf16(h[4 * j + 2], h[4 * j + 3])};
    };
    // the same of g or u alone, in f32 (twice as many pieces)
    auto put_f32 = [&](auto pieces, int row0, int block, const f32x16_t& x) {
        int lane_e = lane;
        asm volatile("" : "+v"(lane_e));
#pragma unroll
        for (int j = 0; j < 4; ++j)
            *(__attribute__((address_space(3))) f32x4_t*)(mine + place(pieces, row0 + (lane_e & 31), block * 8 + j * 2 + (lane_e >> 5))) =
                f32x4_t{x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]};
    };
    auto leave_f32 = [&](auto pieces, float* out, int n_rows, int q0w, int col0) {
        constexpr int K = decltype(pieces)::value;
        const int piece = lane % K, col = p0 + col0 + piece * 4;
        if (col >= a.I) return;
#pragma unroll 4
        for (int i = 0; i < n_rows * K / 64; ++i) {
            const int row = i * (64 / K) + lane / K;
            if (q0w + row >= r.rows) break;
            *reinterpret_cast<f32x4_t*>(out + (int64_t)(r.row0 + q0w + row) * a.I + col) =
                *(__attribute__((address_space(3))) f32x4_t*)(mine + place(pieces, row, piece));
        }
    };
    // the wavefront's rows, the tile's from q0w on, at its columns from col0 on
    auto leave = [&](auto pieces, int n_rows, int q0w, int col0) {
        constexpr int K = decltype(pieces)::value;
        uint16_t* out;
        int64_t pitch;
        int rows, cols;
        if constexpr (MODE == FORWARD) {
            out = a.h + (int64_t)r.row0 * a.I + p0;
            pitch = a.I; rows = r.rows; cols = a.I - p0;
        } else if constexpr (MODE == DROWS) {
            out = a.dx + (int64_t)r.row0 * a.H + p0;
            pitch = a.H; rows = r.rows; cols = a.H - p0;
        } else {
            out = (which ? a.dwu : a.dwg) + ((int64_t)r.expert * a.I + q0) * a.H + p0;
            pitch = a.H; rows = a.I - q0; cols = a.H - p0;
        }
        const int piece = lane % K, col = col0 + piece * 8;
        if (col >= cols) return;
#pragma unroll 4
        for (int i = 0; i < n_rows * K / 64; ++i) {
            const int row = i * (64 / K) + lane / K;
            if (q0w + row >= rows) break;
            *reinterpret_cast<u32x4*>(out + (q0w + row) * pitch + col) =
                *(__attribute__((address_space(3))) u32x4*)(mine + place(pieces, row, piece));
        }
    };
    auto clear = [](auto& acc, int n_p, int n_q) {
#pragma unroll
        for (int t = 0; t < n_p; ++t)
#pragma unroll
            for (int n = 0; n < n_q; ++n)
#pragma unroll
                for (int v = 0; v < 16; ++v) acc[t][n][v] = 0.0f;
    };
    InnerFragment fq_in;
    if (light) {
        if constexpr (MODE != DWEIGHTS) {
            // wavefront w: rows 32 (w / 4) .. + 31, columns 32 (w % 4) .. (FORWARD) or 64 (w % 4) .. + 63
            const int block = wave & 3, row0 = (wave >> 2) * 32;
            InnerLoader<1> lx;
            lx.init(lane, MODE == FORWARD ? a.ldx : a.I, wave * 8);
            lx.piece ^= (wave & 1) * 32;
            auto load_light = [&](int s, char* Q) { load_q_by(lx, s, Q); };
            fq_in.init(lane, wave >> 2);
            f32x16_t acc[2][1];
            clear(acc, 2, 1);
            if constexpr (MODE == FORWARD) {
                InnerFragment fp;
                fp.init(lane, (block >> 1) * 4 + (block & 1));
                multiply_light_stages<2>(stages, P0, P1, P2, Q0, Q1, load_p, load_light, fp, fq_in, acc);
                __syncthreads();
                constexpr std::integral_constant<int, 4> kPieces{};
                if (a.g) {
                    constexpr std::integral_constant<int, 8> kWide{};
                    put_f32(kWide, 0, 0, acc[0][0]);
                    leave_f32(kWide, a.g, 32, row0, block * 32);
                    put_f32(kWide, 0, 0, acc[1][0]);
                    leave_f32(kWide, a.u, 32, row0, block * 32);
                }
                put(kPieces, 0, 0, acc[0][0], acc[1][0]);
                leave(kPieces, 32, row0, block * 32);
            } else {
                OuterFragment<2> fp;
                fp.init(lane, block * 2);
                multiply_light_stages<1>(stages, P0, P1, P2, Q0, Q1, load_p, load_light, fp, fq_in, acc);
                __syncthreads();
                constexpr std::integral_constant<int, 8> kPieces{};
                put(kPieces, 0, 0, acc[0][0], acc[0][0]);
                put(kPieces, 0, 1, acc[1][0], acc[1][0]);
                leave(kPieces, 32, row0, block * 64);
            }
        }
    } else if (wq * 64 < (MODE == DWEIGHTS ? a.I - q0 : r.rows)) {
        f32x16_t acc[4][2];
        clear(acc, 4, 2);
        if constexpr (MODE == FORWARD) {
            InnerFragment fp;
            fp.init(lane, wp * 4);
            fq_in.init(lane, wq * 2);
            multiply_stages(stages, P0, P1, P2, Q0, Q1, load_p, load_q, fp, fq_in, acc);
        } else {
            OuterFragment<4> fp;
            OuterFragment<2> fq_out;
            fp.init(lane, wp * 4);
            if constexpr (MODE == DROWS) {
                fq_in.init(lane, wq * 2);
                multiply_stages(stages, P0, P1, P2, Q0, Q1, load_p, load_q, fp, fq_in, acc);
            } else {
                fq_out.init(lane, wq * 2);
                multiply_stages(stages, P0, P1, P2, Q0, Q1, load_p, load_q, fp, fq_out, acc);
            }
        }
        __syncthreads();
        constexpr int kTiles = MODE == FORWARD ? 2 : 4;
        constexpr std::integral_constant<int, kTiles * 4> kPieces{};
        if constexpr (MODE == FORWARD) {
            if (a.g) {
                constexpr std::integral_constant<int, 16> kWide{};
#pragma unroll
                for (int of = 0; of < 2; ++of) {
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int t = 0; t < 2; ++t) put_f32(kWide, n * 32, t, acc[2 * of + t][n]);
                    leave_f32(kWide, of ? a.u : a.g, 64, wq * 64, wp * 64);
                }
            }
        }
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
                put(kPieces, n * 32, t, acc[t][n], acc[MODE == FORWARD ? t + 2 : t][n]);
        leave(kPieces, 64, wq * 64, wp * kTiles * 32);
    } else {
        load_stages(stages, P0, P1, P2, Q0, Q1, load_p, load_q);
        __syncthreads();
    }
}

// ---------------------------------------------------------------- DWEIGHTS
// P = columns of X, Q = rows of dW (columns of dg or du), inner dimension the expert's rows.  An expert has a
// few stages only, and 128 KB of output per tile: a workgroup per tile spends as long on its beginning and
// its end as on the product.  So there is one workgroup per CU, which takes tile after tile: during a tile's last
// stages the next tile's first ones are on their way, and the output leaves while the next tile begins,
// through 2 KB of LDS of every wavefront's own.  A tile has a multiple of four stages (zeros where there are
// no rows).  Experts differ in rows, so the tiles are given out by a counter per XCD (which workgroup computes
// a tile changes nothing in it); the counter is asked three tiles ahead.  128 experts of 64 rows at 2048 x 768 are
// written at 4.7 TB/s, the rate of a copy (172 us, 218 with a workgroup per tile); where there is more to multiply the
// stores of all CUs come at the same time, and a tile's fourth stage waits for them.
__global__ __launch_bounds__(512) void gated_dweights_kernel(GatedArgs a, int p_tiles, int q_tiles, int* counters) {
    using namespace forge;
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    constexpr int kShortBytes = kTile * kShort * 2;
    __shared__ __attribute__((aligned(1024))) char P0[kShortBytes], P1[kShortBytes], P2[kShortBytes], P3[kShortBytes],
        Q0[kShortBytes], Q1[kShortBytes], Q2[kShortBytes], Q3[kShortBytes], S[8 * 2048];
    __shared__ int slot[2];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wp = wave >> 2, wq = wave & 3;
    // Every XCD takes an eighth of every expert's tiles: those of up to 4 tiles of Q by some of P, which share
    // their panels in its L2 (by 8 or 16 of Q a panel is met again too late: 541 against 528 us with 8168 rows of
    // 16 experts).  Q counts the gate's tiles, then the up projection's.
    const int tiles = p_tiles * q_tiles, per = (tiles + 7) / 8, t0 = (blockIdx.x % 8) * per;
    const int here = min(tiles - t0, per), items = here > 0 ? here * a.E : 0, workers = gridDim.x / 8;
    const int first = blockIdx.x / 8;
    if (first >= items) return;

    typedef __attribute__((address_space(4))) int32_t scalar_int;
    struct Tile {
        int expert, which, p0, q0, row0, rows, stages;
        OuterLoader<kShort> p, q;
    };
    auto tile_at = [&](int item) {
        Tile t;
        t.expert = item / here;
        const int c = t0 + item - t.expert * here, group = c / (4 * p_tiles), in_group = c - group * 4 * p_tiles;
        const int wide = min(q_tiles - group * 4, 4), up_from = (a.I + kTile - 1) / kTile;
        const int q = group * 4 + in_group % wide;
        t.which = q >= up_from;
        t.p0 = in_group / wide * kTile;
        t.q0 = (t.which ? q - up_from : q) * kTile;
        // scalar loads: a vector load would have to wait for the stores before it
        const scalar_int* o = (const scalar_int*)a.offsets + t.expert;
        t.row0 = max(0, min(o[0], a.N));
        t.rows = max(t.row0, min(o[1], a.N)) - t.row0;
        t.stages = max((t.rows + 4 * kShort - 1) / (4 * kShort) * 4, 4);
        t.p.init(wave, lane, a.ldx, a.H - t.p0);
        t.q.init(wave, lane, a.I, a.I - t.q0);
        return t;
    };
    Tile t = tile_at(first), next = t;
    // stage s of tile t; behind its last, the first ones of the next
    auto load = [&](int s, char* P, char* Q) {
        // (selected with a mask: from conditional expressions the compiler makes branches between the products)
        const int on = (t.stages - 1 - s) >> 31;
        auto pick = [&](int mine, int others) { return mine ^ ((mine ^ others) & on); };
        const int k = (s - (t.stages & on)) * kShort, left = pick(t.rows, next.rows) - k;
        const int64_t row = pick(t.row0, next.row0) + k;
        const int p0 = pick(t.p0, next.p0), q0 = pick(t.q0, next.q0);
        OuterLoader<kShort> p, q;
        p.even = pick(t.p.even, next.p.even);
        p.odd = pick(t.p.odd, next.p.odd);
        q.even = pick(t.q.even, next.q.even);
        q.odd = pick(t.q.odd, next.q.odd);
        const int64_t dudg = (const char*)a.du - (const char*)a.dg;
        const uint16_t* grad = (const uint16_t*)((const char*)a.dg + (dudg & -(int64_t)pick(t.which, next.which)));
        p.stage(a.x + row * a.ldx + p0, a.ldx, left, a.H - p0, P, wave);
        q.stage(grad + row * a.I + q0, a.I, left, a.I - q0, Q, wave);
    };
    OuterFragment<4> fp;
    OuterFragment<2> fq;
    fp.init(lane, wp * 4);
    fq.init(lane, wq * 2);
    f32x16_t acc[4][2];
    auto clear = [&] {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int v = 0; v < 16; ++v) acc[t][n][v] = 0.0f;
    };
    load(0, P0, Q0);
    load(1, P1, Q1);
    load(2, P2, Q2);
    load(3, P3, Q3);
    wait_loads_barrier<0>();                                      // all four: no stores are behind their loads yet
    Fragments<4> f;
    f.read(P0, Q0, fp, fq, 0);
    clear();
    constexpr int kStores = 16;
    int coming = first + workers;                                 // the tile after this one
    for (int turn = 0;; ++turn) {
        // asked for now, looked at behind the tile: the third one from here (the sum would wait for the answer)
        int count = 0, opaque = 0;
        asm volatile("" : "+v"(opaque));                          // else the compiler adds up over lanes, and waits
        if (counters && threadIdx.x == 0)
            count = __hip_atomic_fetch_add(counters + blockIdx.x % 8 + opaque, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const bool more = coming < items;
        next = tile_at(more ? coming : first);
        if (!more) next.rows = 0;                                 // zeros, which nobody reads
        // the stores of the tile before are younger than the loads of this one's first four stages
        one_short_stage<8 + kStores>(P0, Q0, P1, Q1, [&] { load(4, P0, Q0); }, fp, fq, f, acc);
        one_short_stage<8 + kStores>(P1, Q1, P2, Q2, [&] { load(5, P1, Q1); }, fp, fq, f, acc);
        one_short_stage<8 + kStores>(P2, Q2, P3, Q3, [&] { load(6, P2, Q2); }, fp, fq, f, acc);
        one_short_stage<8>(P3, Q3, P0, Q0, [&] { load(7, P3, Q3); }, fp, fq, f, acc);
        for (int s = 4; s < t.stages; s += 4) {
            one_short_stage<8>(P0, Q0, P1, Q1, [&] { load(s + 4, P0, Q0); }, fp, fq, f, acc);
            one_short_stage<8>(P1, Q1, P2, Q2, [&] { load(s + 5, P1, Q1); }, fp, fq, f, acc);
            one_short_stage<8>(P2, Q2, P3, Q3, [&] { load(s + 6, P2, Q2); }, fp, fq, f, acc);
            one_short_stage<8>(P3, Q3, P0, Q0, [&] { load(s + 7, P3, Q3); }, fp, fq, f, acc);
        }

        // 32 rows of Q by 32 columns of P at a time: [row][64 bytes], 16-byte piece c of row q at c ^ (q / 4 % 4).
        // Outside the matrix the stores are out of the descriptor's range: all are issued, as counted above.
        uint16_t* out = (t.which ? a.dwu : a.dwg) + ((int64_t)t.expert * a.I + t.q0) * a.H + t.p0;
        const int rows = min(a.I - t.q0, kTile), cols = a.H - t.p0;
        const __amdgpu_buffer_rsrc_t d = descriptor(out, (uint32_t)(((rows - 1) * (int64_t)a.H + min(cols, kTile)) * 2));
        lds_char* mine = (lds_char*)S + wave * 2048;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                int lane_e = lane;
                asm volatile("" : "+v"(lane_e));                  // addresses are formed here, not before the loop
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const f32x16_t& v = acc[b][n];
                    *(__attribute__((address_space(3))) u32x2*)(mine + (lane_e & 31) * 64 + ((j ^ ((lane_e >> 2) & 3)) * 16) + (lane_e >> 5) * 8) =
                        u32x2{pack_bf16(v[4 * j], v[4 * j + 1]), pack_bf16(v[4 * j + 2], v[4 * j + 3])};
                }
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int q = r * 16 + (lane_e >> 2), c = lane_e & 3;
                    const u32x4 v = *(__attribute__((address_space(3))) u32x4*)(mine + q * 64 + ((c ^ ((q >> 2) & 3)) * 16));
                    const int col = wp * 128 + b * 32 + c * 8, row = wq * 64 + n * 32 + q;
                    __builtin_amdgcn_raw_buffer_store_b128(v, d, col < cols && row < rows ? (int)((row * (int64_t)a.H + col) * 2) : (int)kOutside, 0, 0);
                }
            }
        __builtin_amdgcn_sched_barrier(0);
        if (!more) break;
        clear();
        t = next;
        // what was asked for a tile ago was written before a barrier of this tile's
        coming = turn ? __builtin_amdgcn_readfirstlane(slot[(turn - 1) & 1]) : first + 2 * workers;
        if (threadIdx.x == 0) slot[turn & 1] = counters ? 3 * workers + count : first + (turn + 3) * workers;
    }
    // loads of zeros are still on their way to LDS: a workgroup that ends gives its LDS away
    wait_loads<0>();
}

// ---------------------------------------------------------------- few rows: FORWARD alone
// Bound by the weights of the experts that have rows, which stream through once.  A wavefront takes 16
// features (their rows of Wg and of Wu) and every `split`-th run of 128 columns, and no barrier
// before the end; the split wavefronts that share their features add up in LDS in a fixed order.
// A workgroup's 8 wavefronts cover 128 / split features: the host splits as far as it takes to fill
// the GPU, and no further, since a wavefront with few runs spends its time on its beginning and end.
// Every wavefront has two LDS buffers of its own, one run each.  Runs go there by loads of 256
// consecutive bytes of 4 rows (straight into registers the matrix instruction's layout would fetch 64
// bytes of 16 rows at a time, which HBM serves a third slower); 16-byte piece c of row n lies at c ^ n.
// MT blocks of 16 rows, which come from the caches.  8 experts of one row, 7168 x 2048: 80 us, 5.8 TB/s, what pure
// reads reach on this card.
constexpr int kRunBytes = 32 * 256;                              // 16 rows of Wg, 16 of Wu, 128 columns
template <int MT>
__global__ __launch_bounds__(512) void gated_few_kernel(GatedArgs a, int p_tiles, int split) {
    using namespace forge;
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    __shared__ __attribute__((aligned(1024))) char S0[8 * kRunBytes], S1[8 * kRunBytes];
    __shared__ FindSlot slot;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, kb = lane >> 4;
    const int share = wave % split;                              // which of its features' runs
    RaggedTile r;
    if (!find_tile(a.offsets, a.E, a.N, 16 * MT, 0, p_tiles, [](int, int) { return (int)blockIdx.x; }, r, slot)) return;
    const int f0 = r.p * (128 / split), i0 = f0 + wave / split * 16;
    const int inner = r.expert < 0 ? 0 : a.H;
    const int wrows = min(a.I - i0, 16);                          // none for a wavefront behind the last feature
    const int64_t we = (int64_t)(r.expert < 0 ? 0 : r.expert) * a.ws + (wrows > 0 ? (int64_t)i0 * a.ldw : 0);
    const uint32_t wbytes = wrows > 0 ? (uint32_t)(((wrows - 1) * a.ldw + a.H) * 2) : 0u;
    const __amdgpu_buffer_rsrc_t dg = descriptor(a.wg + we, wbytes), du = descriptor(a.wu + we, wbytes);
    const __amdgpu_buffer_rsrc_t dx = descriptor(a.x + (int64_t)r.row0 * a.ldx, (uint32_t)(((r.rows - 1) * a.ldx + a.H) * 2));
    f32x4_t g[MT], u[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) g[t] = u[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    const int runs = (inner + 127) / 128;
    // (weight rows and rows behind the last are beyond their descriptors)
    auto fetch = [&](int c, char* S, u32x4 (&x)[MT][4]) {
        char* to = S + wave * kRunBytes;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int row = j * 4 + kb, k = c * 128 + (n ^ row) * 8;
            const uint32_t at = k < inner ? (uint32_t)((row * a.ldw + k) * 2) : kOutside;
            load_to_lds(dg, to + j * 1024, at);
            load_to_lds(du, to + 4096 + j * 1024, at);
        }
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const int k = c * 128 + d * 32 + kb * 8;
                x[t][d] = __builtin_amdgcn_raw_buffer_load_b128(
                    dx, k < inner ? (int)(((t * 16 + n) * a.ldx + k) * 2) : (int)kOutside, 0, 0);
            }
        __builtin_amdgcn_sched_barrier(0);
    };
    auto multiply = [&](const char* S, const u32x4 (&x)[MT][4]) {
        const char* from = S + wave * kRunBytes + n * 256;
        bf16x8_t wg[4], wu[4];
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            wg[d] = *reinterpret_cast<const bf16x8_t*>(from + (((d * 4 + kb) ^ n) * 16));
            wu[d] = *reinterpret_cast<const bf16x8_t*>(from + 4096 + (((d * 4 + kb) ^ n) * 16));
        }
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const bf16x8_t xv = __builtin_bit_cast(bf16x8_t, x[t][d]);
                g[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wg[d], xv, g[t], 0, 0, 0);
                u[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wu[d], xv, u[t], 0, 0, 0);
            }
        // the buffer is free once the reads are back
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(0xC07F);                       // lgkmcnt(0)
        __builtin_amdgcn_sched_barrier(0);
    };
    // all but the last run's loads (8 to LDS, 4 MT to registers) have arrived
    auto arrived = [] {
        constexpr int kLater = 8 + 4 * MT;
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(0x0F70 | (kLater & 15) | ((kLater >> 4) << 14));
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
    };
    u32x4 x0[MT][4], x1[MT][4];
    // runs behind the last are fetched as zeros, so that every wavefront always has two on their way
    fetch(share, S0, x0);
    fetch(share + split, S1, x1);
    for (int c = share; c < runs; c += 2 * split) {
        arrived();
        multiply(S0, x0);
        fetch(c + 2 * split, S0, x0);
        arrived();
        multiply(S1, x1);
        fetch(c + 3 * split, S1, x1);
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);                           // vmcnt(0): the zeros behind the last run
    __syncthreads();
    // [wavefront][block of rows][gate, up][row][feature]; register v: feature 4 (lane / 16) + v, row lane & 15
    float* part = reinterpret_cast<float*>(S0);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        *reinterpret_cast<f32x4_t*>(part + ((wave * MT + t) * 2 + 0) * 256 + n * 16 + kb * 4) = g[t];
        *reinterpret_cast<f32x4_t*>(part + ((wave * MT + t) * 2 + 1) * 256 + n * 16 + kb * 4) = u[t];
    }
    __syncthreads();
    const int features = 128 / split;
    for (int o = threadIdx.x; o < MT * 16 * features; o += 512) {
        const int q = o / features, f = o % features;
        if (q >= r.rows || f0 + f >= a.I) continue;
        const float* p = part + ((f / 16 * split * MT + q / 16) * 2) * 256 + (q % 16) * 16 + f % 16;
        float gs = 0.0f, us = 0.0f;
        for (int w = 0; w < split; ++w, p += MT * 512) {
            gs += p[0];
            us += p[256];
        }
        const int64_t at = (int64_t)(r.row0 + q) * a.I + f0 + f;
        a.h[at] = f32_to_bf16_bits(act_f32(a.act, gs) * us);
        if (a.g) {
            a.g[at] = gs;
            a.u[at] = us;
        }
    }
}

// ---------------------------------------------------------------- few rows: DROWS
// The same idea with W's rows as the inner dimension: a workgroup takes 128 columns of X and one tile
// of 32 rows, its 8 wavefronts every eighth run of 32 of W's rows (the gate's, then the up
// projection's), 256 consecutive bytes of each, and their sums meet in LDS in a fixed order.  H / 128
// workgroups of 2 I / 256 runs per expert where the tiles above have H / 256 of 2 I / 64 stages.
// A run's row k lies at 256 k, its 16-byte piece c at c ^ 4 (k % 4): transposed reads as in mfma_tile.h.
// One expert of 64 rows, 7168 x 2048 (59 MB): 30 us.
__global__ __launch_bounds__(512) void gated_drows_few_kernel(GatedArgs a, int p_tiles) {
    using namespace forge;
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    constexpr int kRun = 32 * 256;
    __shared__ __attribute__((aligned(1024))) char S0[8 * kRun], S1[8 * kRun];
    __shared__ FindSlot slot;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    RaggedTile r;
    if (!find_tile(a.offsets, a.E, a.N, 32, 0, p_tiles, [](int, int) { return (int)blockIdx.x; }, r, slot)) return;
    const int p0 = r.p * 128;
    const int per_phase = r.expert < 0 ? 0 : (a.I + 31) / 32, runs = 2 * per_phase;
    const int64_t we = (int64_t)(r.expert < 0 ? 0 : r.expert) * a.ws + p0;
    const int cols = min(a.H - p0, 128);
    // this lane's place in a load of 4 rows
    const int row = lane >> 4, piece = (lane & 15) ^ (row << 2);
    const uint32_t at0 = piece * 8 < cols ? (uint32_t)((row * a.ldw + piece * 8) * 2) : kOutside;
    auto fetch = [&](int c, char* S, u32x4 (&q)[2]) {
        const bool up = c >= per_phase;
        const int k0 = (up ? c - per_phase : c) * 32;
        // runs behind the last have no rows: zeros
        const int rows = c < runs ? min(a.I - k0, 32) : 0;
        const int size = max((rows - 1) * (int)a.ldw + cols, 0);
        const __amdgpu_buffer_rsrc_t dw = descriptor((up ? a.wu : a.wg) + we + (c < runs ? k0 * a.ldw : 0), (uint32_t)size * 2);
        const __amdgpu_buffer_rsrc_t dd = descriptor((up ? a.du : a.dg) + (int64_t)r.row0 * a.I, (uint32_t)(r.rows * a.I * 2));
#pragma unroll
        for (int j = 0; j < 8; ++j) load_to_lds(dw, S + wave * kRun + j * 1024, at0 + (uint32_t)(j * 8 * a.ldw));
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int k = k0 + s * 16 + (lane >> 5) * 8;
            q[s] = __builtin_amdgcn_raw_buffer_load_b128(
                dd, c < runs && k < a.I ? (int)(((lane & 31) * a.I + k) * 2) : (int)kOutside, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    f32x16_t acc[4];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[t][v] = 0.0f;
    uint32_t from[4];
    {
        const int g = lane >> 4, i = lane & 15, k = 8 * (g >> 1) + (i >> 2), col = 16 * (g & 1) + 4 * (i & 3);
#pragma unroll
        for (int t = 0; t < 4; ++t) from[t] = wave * kRun + k * 256 + ((((col >> 3) + t * 4) ^ ((i >> 2) << 2)) * 16) + (col & 7) * 2;
    }
    auto multiply = [&](const char* S, const u32x4 (&q)[2]) {
        typedef short s16x8 __attribute__((ext_vector_type(8)));
        bf16x8_t p[2][4];
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const char* f = S + from[t] + s * 4096;
                const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)f);
                const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(f + 1024));
                const s16x8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                p[s][t] = __builtin_bit_cast(bf16x8_t, v);
            }
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int t = 0; t < 4; ++t)
                acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(p[s][t], __builtin_bit_cast(bf16x8_t, q[s]), acc[t], 0, 0, 0);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(0xC07F);                       // lgkmcnt(0): the buffer is free
        __builtin_amdgcn_sched_barrier(0);
    };
    auto arrived = [] {                                           // all but the last run's 10 loads
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(0x0F7A);
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
    };
    u32x4 q0[2], q1[2];
    fetch(wave, S0, q0);
    fetch(wave + 8, S1, q1);
    for (int c = wave; c < runs; c += 16) {
        arrived();
        multiply(S0, q0);
        fetch(c + 16, S0, q0);
        arrived();
        multiply(S1, q1);
        fetch(c + 24, S1, q1);
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);
    __syncthreads();
    // [wavefront][row][128 columns] f32, 16 KB a wavefront: four in either buffer.  Registers 4 j .. 4 j + 3
    // of tile t: columns 32 t + 8 j + 4 (lane / 32) .. + 3, row lane & 31; 16-byte piece c of row q at c ^ q.
    {
        char* part = (wave < 4 ? S0 : S1) + (wave & 3) * 16384 + (lane & 31) * 512;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f32x4_t v;
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = acc[t][4 * j + i];
                *reinterpret_cast<f32x4_t*>(part + (((t * 8 + j * 2 + (lane >> 5)) ^ (lane & 31)) * 16)) = v;
            }
    }
    __syncthreads();
    // a thread sums 4 columns of one row, twice
    for (int o = threadIdx.x; o < 32 * 32; o += 512) {
        const int q = o >> 5, c = o & 31;
        if (q >= r.rows || c * 4 >= cols) continue;
        f32x4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < 8; ++w)
            v += *reinterpret_cast<const f32x4_t*>((w < 4 ? S0 : S1) + (w & 3) * 16384 + q * 512 + ((c ^ q) * 16));
        *reinterpret_cast<uint2*>(a.dx + (int64_t)(r.row0 + q) * a.H + p0 + c * 4) =
            make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
    }
}

// dg and du from g, u and dh, rounded to bf16 once (they are operands of the two products), 8 elements
// per thread: 14 bytes moved per element; 8168 x 2048 (234 MB, of which the last level cache holds a part) 36 us
__global__ __launch_bounds__(256) void gated_grad_kernel(const uint4* __restrict__ dh,
                                                          const f32x4_t* __restrict__ g,
                                                          const f32x4_t* __restrict__ u, uint4* __restrict__ dg,
                                                          uint4* __restrict__ du, int64_t n8, int act, int* __restrict__ counters) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < 8) counters[i] = 0;                                   // for the launch behind this one
    if (i >= n8) return;
    const uint4 d4 = dh[i];
    const f32x4_t gv[2] = {g[2 * i], g[2 * i + 1]}, uv[2] = {u[2 * i], u[2 * i + 1]};
    const uint32_t dw[4] = {d4.x, d4.y, d4.z, d4.w};
    uint32_t og[4], ou[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float x[2], y[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const float d = __uint_as_float(k ? dw[j] & 0xFFFF0000u : dw[j] << 16);
            float va, vd;
            act_grad_f32(act, gv[j / 2][2 * (j & 1) + k], va, vd);
            x[k] = d * uv[j / 2][2 * (j & 1) + k] * vd;
            y[k] = d * va;
        }
        og[j] = pack_bf16(x[0], x[1]);
        ou[j] = pack_bf16(y[0], y[1]);
    }
    dg[i] = make_uint4(og[0], og[1], og[2], og[3]);
    du[i] = make_uint4(ou[0], ou[1], ou[2], ou[3]);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

constexpr int64_t kFillWorkgroups = 256;
// The kernels for few rows rather than the tiles: where there are few rows in all, and where the tiles would not
// fill the GPU.  Weights from HBM, us, few against tiles:
//   forward, 7168 x 2048: one expert of 64 rows 33 / 96, of 256 88 / 180; 8 experts of 8 rows 136 / 149, of 32 144 /
//     150, of 64 173 / 153; 32 experts of 4 rows 372 / 372, of 32 420 / 374
//   forward, 2048 x 768: 8 experts of 32 rows 28 / 31, of 64 40 / 33; 32 of 8 rows 58 / 64, of 32 73 / 67; 128 of 2
//     rows 209 / 216, of 4 206 / 200, of 64 291 / 208
//   d rows, 7168 x 2048: one expert of 64 rows 30 / 39, of 256 78 / 82; 8 experts of 8 rows 87 / 80
//   d rows, 2048 x 768: one expert of 256 rows 16 / 35; 8 of 8 rows 15 / 19, of 64 23 / 20; 32 of 8 rows 38 / 35
bool few_rows(int64_t N, int64_t E, int64_t I) {
    return N <= 256 || (N <= 32 * E && E * forge::ceil_div(I, 128) < kFillWorkgroups);
}
bool few_rows_back(int64_t N, int64_t E, int64_t H) {
    return N <= 256 && (N < E ? N : E) * forge::ceil_div(H, 256) <= kFillWorkgroups / 2;
}
// and how many rows of x per workgroup (8 experts of 16 rows: 98 with 16, 101 with 32, 116 with 64;
// of 64 rows: 238, 178, 152)
int few_tile(int64_t N, int64_t E) { return N <= 32 || N <= 16 * E ? 16 : N <= 64 || N <= 48 * E ? 32 : 64; }

// From so many rows per expert on a workgroup per tile does better than one per CU (gated_dweights_kernel), whose
// stages are fetched less far ahead: 7168 x 2048, us, per CU against per tile: 16 experts of 64 rows 212 / 256, 16
// with 8168 rows by popularity 528 / 630, of 1024 rows 905 / 975, 8 of 2048 rows 831 / 811, 4 of 4096 rows 790 / 742,
// one of 8192 411 / 365
constexpr int64_t kLongExperts = 2048;

int64_t grad_bytes(int64_t N, int64_t I) { return forge::ceil_div(2 * N * I, 256) * 256; }

// out[b][r][c] = in[b][r][c], zeros behind the last row and column; 8 elements per thread, bound by HBM.  Rows start
// anywhere: an odd element's 16 bytes are put together from the five 4-byte words they lie across.
__global__ __launch_bounds__(256) void pad_rows_kernel(const uint16_t* __restrict__ in, int64_t stride, int64_t ld,
                                                       uint4* __restrict__ out, int R, int C, int Rp, int Cp8,
                                                       const int32_t* __restrict__ offsets) {
    const int b = blockIdx.y;
    if (offsets && offsets[b] >= offsets[b + 1]) return;         // nobody reads this one
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)Rp * Cp8) return;
    const int r = (int)(i / Cp8), c = (int)(i - (int64_t)r * Cp8) * 8;
    uint32_t v[4] = {0, 0, 0, 0};
    if (r < R && c < C) {
        const uint16_t* p = in + b * stride + (int64_t)r * ld + c;
        const bool odd = (reinterpret_cast<uintptr_t>(p) & 2) != 0;
        if (c + 8 <= C && !odd) {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = reinterpret_cast<const uint32_t*>(p)[j];
        } else if (c > 0 && c + 8 < C) {                          // the words' other halves are the row's own
            const uint32_t* q = reinterpret_cast<const uint32_t*>(p - 1);
            uint32_t w = q[0];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t next = q[j + 1];
                v[j] = w >> 16 | next << 16;
                w = next;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c + j < C) v[j / 2] |= (uint32_t)p[j] << (16 * (j & 1));
        }
    }
    out[(int64_t)b * Rp * Cp8 + i] = make_uint4(v[0], v[1], v[2], v[3]);
}

int check(const char* name, const void* rows, int64_t ldx, const int32_t* offsets, const void* Wg,
          const void* Wu, int64_t ldw, int64_t w_stride, int64_t N, int64_t E, int64_t H, int64_t I, int act) {
    FORGE_REQUIRE(N >= 0 && E >= 1 && H >= 1 && I >= 1, "%s: N=%lld E=%lld H=%lld I=%lld", name, (long long)N,
                  (long long)E, (long long)H, (long long)I);
    FORGE_REQUIRE(N <= (1 << 30) && E <= 65535 && H < (1 << 21) && I < (1 << 21) && ldx < (1 << 21) && ldw < (1 << 21),
                  "%s: N=%lld E=%lld H=%lld I=%lld: too large (N up to 2^30, E below 2^16, H, I and the row pitches below 2^21)",
                  name, (long long)N, (long long)E, (long long)H, (long long)I);
    FORGE_REQUIRE(act >= FORGE_ACT_NONE && act <= FORGE_ACT_RELU, "%s: act=%d", name, act);
    FORGE_REQUIRE(offsets && Wg && Wu && (rows || N == 0), "%s: null pointer", name);
    FORGE_REQUIRE(ldx >= H && ldw >= H && (E == 1 || w_stride >= I * ldw),
                  "%s: row pitch %lld / %lld below H=%lld or expert stride %lld below I rows", name,
                  (long long)ldx, (long long)ldw, (long long)H, (long long)w_stride);
    FORGE_REQUIRE(H % 8 == 0 && I % 8 == 0 && ldx % 8 == 0 && ldw % 8 == 0 && (E == 1 || w_stride % 8 == 0) &&
                      aligned16(rows) && aligned16(Wg) && aligned16(Wu),
                  "%s: H=%lld, I=%lld, pitches and strides must be multiples of 8 elements and pointers 16-byte aligned "
                  "(forge_pad_rows makes such copies)", name, (long long)H, (long long)I);
    return FORGE_OK;
}
}  // namespace

extern "C" int forge_pad_rows(const void* in, int64_t stride, int64_t ld, void* out, int64_t batch, int64_t R,
                              int64_t C, int64_t Rp, int64_t Cp, const int32_t* offsets, forge_stream_t stream) {
    const char* name = "forge_pad_rows";
    FORGE_REQUIRE(batch >= 0 && R >= 0 && C >= 1 && Rp >= R && Cp >= C && Cp % 8 == 0,
                  "%s: batch=%lld R=%lld C=%lld Rp=%lld Cp=%lld", name, (long long)batch, (long long)R, (long long)C,
                  (long long)Rp, (long long)Cp);
    FORGE_REQUIRE(batch <= 65535 && Rp < (1 << 30) && Cp < (1 << 24) && forge::ceil_div(Rp * Cp / 8, 256) <= forge::max_workgroups(256),
                  "%s: batch=%lld Rp=%lld Cp=%lld: too large", name, (long long)batch, (long long)Rp, (long long)Cp);
    if (batch == 0 || Rp == 0) return FORGE_OK;
    FORGE_REQUIRE(in && out, "%s: null pointer", name);
    FORGE_REQUIRE(aligned16(out) && (reinterpret_cast<uintptr_t>(in) & 1) == 0, "%s: out not 16-byte aligned", name);
    FORGE_REQUIRE(ld >= C, "%s: row pitch %lld below C=%lld", name, (long long)ld, (long long)C);
    hipStream_t st = (hipStream_t)stream;
    forge::KernelTiming timing("pad_rows", st, 2.0 * batch * (R * C + Rp * Cp), forge::WORK_BYTES);
    pad_rows_kernel<<<dim3((unsigned)forge::ceil_div(Rp * Cp / 8, 256), (unsigned)batch), 256, 0, st>>>(
        (const uint16_t*)in, stride, ld, (uint4*)out, (int)R, (int)C, (int)Rp, (int)(Cp / 8), offsets);
    FORGE_LAUNCH_CHECK();
    return FORGE_OK;
}

extern "C" int forge_gated_rows(const void* rows, int64_t ldx, const int32_t* offsets, const void* Wg,
                                const void* Wu, int64_t ldw, int64_t w_stride, int64_t N, int64_t E,
                                int64_t H, int64_t I, int act, void* h, float* gate_out, float* up_out,
                                forge_stream_t stream) {
    const char* name = "forge_gated_rows";
    if (int rc = check(name, rows, ldx, offsets, Wg, Wu, ldw, w_stride, N, E, H, I, act)) return rc;
    if (N == 0) return FORGE_OK;
    FORGE_REQUIRE(h, "%s: null pointer", name);
    FORGE_REQUIRE((gate_out == nullptr) == (up_out == nullptr), "%s: gate_out and up_out go together", name);
    FORGE_REQUIRE(aligned16(h) && aligned16(gate_out) && aligned16(up_out), "%s: outputs not 16-byte aligned", name);
    GatedArgs a{};
    a.x = (const uint16_t*)rows; a.offsets = offsets; a.wg = (const uint16_t*)Wg; a.wu = (const uint16_t*)Wu;
    a.ldx = ldx; a.ldw = ldw; a.ws = w_stride;
    a.N = (int)N; a.E = (int)E; a.H = (int)H; a.I = (int)I; a.act = act;
    a.h = (uint16_t*)h; a.g = gate_out; a.u = up_out;
    hipStream_t st = (hipStream_t)stream;
    forge::KernelTiming timing("gated_rows", st, 4.0 * N * H * I, forge::WORK_FLOPS);
    const bool few = few_rows(N, E, I);
    const int64_t live = N < E ? N : E;                           // experts with rows, at most
    int split = 1;
    while (few && split < 8 && forge::ceil_div(I, 128 / split) * live < kFillWorkgroups) split *= 2;
    const int64_t p_tiles = forge::ceil_div(I, few ? 128 / split : 128);
    const int q_tile = few ? few_tile(N, E) : 256;
    const int64_t blocks = forge::ceil_div(p_tiles * forge::ragged_tiles(N, E, q_tile), 8) * 8 + 8;
    FORGE_REQUIRE(blocks <= forge::max_workgroups(512), "%s: %lld workgroups, too many for one launch", name, (long long)blocks);
    const dim3 grid((unsigned)blocks);
    if (!few) gated_tile_kernel<FORWARD><<<grid, 512, 0, st>>>(a, (int)p_tiles, 1);
    else if (q_tile == 16) gated_few_kernel<1><<<grid, 512, 0, st>>>(a, (int)p_tiles, split);
    else if (q_tile == 32) gated_few_kernel<2><<<grid, 512, 0, st>>>(a, (int)p_tiles, split);
    else gated_few_kernel<4><<<grid, 512, 0, st>>>(a, (int)p_tiles, split);
    FORGE_LAUNCH_CHECK();
    return FORGE_OK;
}

extern "C" int64_t forge_gated_rows_backward_workspace_bytes(int64_t N, int64_t I) {
    return N > 0 && I > 0 ? 2 * grad_bytes(N, I) + 256 : 0;
}

extern "C" int forge_gated_rows_backward(const void* dh, const float* g, const float* u, const void* rows,
                                         int64_t ldx, const int32_t* offsets, const void* Wg, const void* Wu,
                                         int64_t ldw, int64_t w_stride, int64_t N, int64_t E, int64_t H,
                                         int64_t I, int act, void* drows, void* dWg, void* dWu, void* ws,
                                         int64_t ws_bytes, forge_stream_t stream) {
    const char* name = "forge_gated_rows_backward";
    if (int rc = check(name, rows, ldx, offsets, Wg, Wu, ldw, w_stride, N, E, H, I, act)) return rc;
    FORGE_REQUIRE(N == 0 || (dh && g && u && ws), "%s: null pointer", name);
    FORGE_REQUIRE(N == 0 || ws_bytes >= forge_gated_rows_backward_workspace_bytes(N, I),
                  "%s: workspace of %lld bytes, %lld needed", name, (long long)ws_bytes,
                  (long long)forge_gated_rows_backward_workspace_bytes(N, I));
    FORGE_REQUIRE(aligned16(ws) && aligned16(dh) && aligned16(g) && aligned16(u) && aligned16(drows) && aligned16(dWg) &&
                      aligned16(dWu), "%s: workspace, gradients, g and u must be 16-byte aligned", name);
    uint16_t* dg = (uint16_t*)ws;
    uint16_t* du = (uint16_t*)((char*)ws + grad_bytes(N, I));
    hipStream_t st = (hipStream_t)stream;
    GatedArgs a{};
    a.x = (const uint16_t*)rows; a.offsets = offsets; a.wg = (const uint16_t*)Wg; a.wu = (const uint16_t*)Wu;
    a.ldx = ldx; a.ldw = ldw; a.ws = w_stride;
    a.N = (int)N; a.E = (int)E; a.H = (int)H; a.I = (int)I; a.act = act;
    a.dg = dg; a.du = du;
    a.dx = (uint16_t*)drows; a.dwg = (uint16_t*)dWg; a.dwu = (uint16_t*)dWu;
    const bool few = few_rows_back(N, E, H);
    const int64_t h_tiles = forge::ceil_div(H, 256), i_tiles = forge::ceil_div(I, 256), p_tiles = few ? forge::ceil_div(H, 128) : h_tiles;
    const int64_t row_blocks = forge::ceil_div(p_tiles * forge::ragged_tiles(N, E, few ? 32 : 256), 8) * 8 + 8;
    FORGE_REQUIRE(row_blocks <= forge::max_workgroups(512) && 16 * forge::ceil_div(h_tiles * i_tiles, 8) * E <= INT32_MAX &&
                      forge::ceil_div(N * I / 8, 256) <= forge::max_workgroups(256),
                  "%s: too many workgroups for one launch", name);
    if (N > 0) {
        forge::KernelTiming timing("gated_grad", st, 14.0 * N * I, forge::WORK_BYTES);
        gated_grad_kernel<<<dim3((unsigned)forge::ceil_div(N * I / 8, 256)), 256, 0, st>>>(
            (const uint4*)dh, (const f32x4_t*)g, (const f32x4_t*)u, (uint4*)dg, (uint4*)du, N * I / 8, act, (int*)((char*)ws + 2 * grad_bytes(N, I)));
        FORGE_LAUNCH_CHECK();
    }
    if (drows && N > 0) {
        forge::KernelTiming timing("gated_drows", st, 4.0 * N * H * I, forge::WORK_FLOPS);
        if (few) gated_drows_few_kernel<<<dim3((unsigned)row_blocks), 512, 0, st>>>(a, (int)p_tiles);
        else gated_tile_kernel<DROWS><<<dim3((unsigned)row_blocks), 512, 0, st>>>(a, (int)p_tiles, 1);
        FORGE_LAUNCH_CHECK();
    }
    if (dWg || dWu) {
        forge::KernelTiming timing("gated_dweights", st, 2.0 * N * H * I * ((dWg ? 1 : 0) + (dWu ? 1 : 0)), forge::WORK_FLOPS);
        // gate weights first, then up weights; one alone is passed as the first
        const int both = dWg && dWu ? 2 : 1;
        if (!dWg) { a.dg = du; a.dwg = a.dwu; }
        if (N >= kLongExperts * E) {
            const int64_t blocks = forge::ceil_div(h_tiles * i_tiles, 8) * 8 * E * both;
            FORGE_REQUIRE(blocks <= forge::max_workgroups(512), "%s: %lld workgroups, too many for one launch", name, (long long)blocks);
            gated_tile_kernel<DWEIGHTS><<<dim3((unsigned)blocks), 512, 0, st>>>(a, (int)h_tiles, (int)i_tiles);
        } else {
            const int64_t items = forge::ceil_div(h_tiles * i_tiles * both, 8) * E;    // of an XCD
            const int64_t blocks = 8 * (items < kFillWorkgroups / 8 ? items : kFillWorkgroups / 8);
            gated_dweights_kernel<<<dim3((unsigned)blocks), 512, 0, st>>>(
                a, (int)h_tiles, (int)(i_tiles * both), N > 0 ? (int*)((char*)ws + 2 * grad_bytes(N, I)) : nullptr);
        }
        FORGE_LAUNCH_CHECK();
    }
    return FORGE_OK;
}
