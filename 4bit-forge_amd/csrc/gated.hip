// Gated feed-forward rows of routed experts and their gradients.
//
//   forward    g = X_e Wg[e]^T,  u = X_e Wu[e]^T,  h = act(g) * u
//   backward   dg = dh * u * act'(g),  du = dh * act(g)
//              dX_e = dg Wg[e] + du Wu[e],  dWg[e] = dg^T X_e,  dWu[e] = du^T X_e
//
// Three products over one ragged batch.  All run on the bf16 matrix instruction with f32 sums.
#include "act.h"
#include "common.h"
#include "ragged.h"

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

// ---------------------------------------------------------------- any shape, any alignment
// 64 x 64 outputs per workgroup, four wavefronts of 32 x 32, 32 of the inner dimension a step
// through LDS, every element loaded by itself under its own bounds: what takes the calls whose
// rows are not 16-byte aligned.
//   FORWARD   P = weight rows (32 of Wg above the same 32 of Wu), Q = rows,         inner H
//   DROWS     P = columns of X, Q = rows,                                           inner I, twice
//   DWEIGHTS  P = columns of X, Q = rows of dW,                                     inner the expert's rows
// P runs along the registers of the accumulator, i.e. along the output's contiguous dimension.
template <int MODE>
__global__ __launch_bounds__(256) void gated_any_kernel(GatedArgs a, int p_tiles) {
    constexpr int T = 64, K = 32, LD = K + 8;
    __shared__ uint16_t P[T][LD], Q[T][LD];
    __shared__ int slot[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wp = wave >> 1, wq = wave & 1;
    const int pt = blockIdx.x % p_tiles, qt = blockIdx.x / p_tiles;

    RaggedTile r;
    int q0 = 0, expert, inner, phases = 1;
    const uint16_t* dgu = nullptr;
    uint16_t* dw = nullptr;
    if constexpr (MODE == DWEIGHTS) {
        const int i_tiles = (a.I + T - 1) / T;
        const int which = blockIdx.z;
        expert = blockIdx.y;
        q0 = qt * T;
        if (qt >= i_tiles) return;
        r.expert = expert;
        r.row0 = forge::clamp_offset(a.offsets, expert, 0, a.N);
        r.rows = forge::clamp_offset(a.offsets, expert + 1, r.row0, a.N) - r.row0;
        inner = r.rows;
        dgu = which ? a.du : a.dg;
        dw = which ? a.dwu : a.dwg;
    } else {
        if (!find_tile(a.offsets, a.E, a.N, T, qt, r, slot)) return;
        expert = r.expert;
        inner = expert < 0 ? 0 : (MODE == FORWARD ? a.H : a.I);
        phases = MODE == DROWS ? 2 : 1;
    }
    const int64_t wbase = (int64_t)(expert < 0 ? 0 : expert) * a.ws;
    const int p0 = pt * (MODE == FORWARD ? T / 2 : T);

    f32x16_t acc;
#pragma unroll
    for (int v = 0; v < 16; ++v) acc[v] = 0.0f;
    for (int ph = 0; ph < phases; ++ph)
        for (int k0 = 0; k0 < inner; k0 += K) {
            __syncthreads();
            for (int i = threadIdx.x; i < T * K; i += 256) {
                // neighbouring threads along whichever index is contiguous in memory
                int row, k;
                if (MODE == FORWARD) { k = i % K; row = i / K; } else { row = i % T; k = i / T; }
                uint16_t v = 0;
                if (k0 + k < inner) {
                    if constexpr (MODE == FORWARD) {
                        const int w = p0 + (row & 31);
                        if (w < a.I) v = (row < 32 ? a.wg : a.wu)[wbase + (int64_t)w * a.ldw + k0 + k];
                    } else if constexpr (MODE == DROWS) {
                        if (p0 + row < a.H) v = (ph ? a.wu : a.wg)[wbase + (int64_t)(k0 + k) * a.ldw + p0 + row];
                    } else {
                        if (p0 + row < a.H) v = a.x[(int64_t)(r.row0 + k0 + k) * a.ldx + p0 + row];
                    }
                }
                P[row][k] = v;
                int qr, qk;
                if (MODE != DWEIGHTS) { qk = i % K; qr = i / K; } else { qr = i % T; qk = i / T; }
                v = 0;
                if (k0 + qk < inner) {
                    if constexpr (MODE == FORWARD) {
                        if (qr < r.rows) v = a.x[(int64_t)(r.row0 + qr) * a.ldx + k0 + qk];
                    } else if constexpr (MODE == DROWS) {
                        if (qr < r.rows) v = (ph ? a.du : a.dg)[(int64_t)(r.row0 + qr) * a.I + k0 + qk];
                    } else {
                        if (q0 + qr < a.I) v = dgu[(int64_t)(r.row0 + k0 + qk) * a.I + q0 + qr];
                    }
                }
                Q[qr][qk] = v;
            }
            __syncthreads();
#pragma unroll
            for (int s = 0; s < K; s += 16) {
                // FORWARD: this wavefront's 32 P rows are 16 of Wg and the same 16 of Wu
                const int pr = MODE == FORWARD ? ((lane & 31) < 16 ? wp * 16 + (lane & 15) : 32 + wp * 16 + (lane & 15))
                                               : wp * 32 + (lane & 31);
                const bf16x8_t pv = *reinterpret_cast<const bf16x8_t*>(&P[pr][s + 8 * (lane >> 5)]);
                const bf16x8_t qv = *reinterpret_cast<const bf16x8_t*>(&Q[wq * 32 + (lane & 31)][s + 8 * (lane >> 5)]);
                acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(pv, qv, acc, 0, 0, 0);
            }
        }
    // register v of the accumulator: row 8 (v >> 2) + 4 (lane >> 5) + (v & 3) of P, column lane & 31 of Q
    const int q = wq * 32 + (lane & 31);
    if constexpr (MODE == FORWARD) {
        if (q >= r.rows) return;
#pragma unroll
        for (int v = 0; v < 8; ++v) {                  // rows 0..15: gate, 16..31: up (registers v and v + 8)
            const int i = p0 + wp * 16 + 8 * (v >> 2) + 4 * (lane >> 5) + (v & 3);
            if (i >= a.I) continue;
            const int64_t at = (int64_t)(r.row0 + q) * a.I + i;
            a.h[at] = f32_to_bf16_bits(act_f32(a.act, acc[v]) * acc[v + 8]);
            if (a.g) {
                a.g[at] = acc[v];
                a.u[at] = acc[v + 8];
            }
        }
    } else {
        if (MODE == DROWS ? q >= r.rows : q0 + q >= a.I) return;
        uint16_t* out = MODE == DROWS ? a.dx + (int64_t)(r.row0 + q) * a.H
                                      : dw + ((int64_t)expert * a.I + q0 + q) * a.H;
#pragma unroll
        for (int v = 0; v < 16; ++v) {
            const int c = p0 + wp * 32 + 8 * (v >> 2) + 4 * (lane >> 5) + (v & 3);
            if (c < a.H) out[c] = f32_to_bf16_bits(acc[v]);
        }
    }
}

// dg and du from g, u and dh, rounded to bf16 once (they are operands of the two products);
// one element per thread
__global__ __launch_bounds__(256) void gated_grad_kernel(const uint16_t* __restrict__ dh,
                                                         const float* __restrict__ g,
                                                         const float* __restrict__ u,
                                                         uint16_t* __restrict__ dg,
                                                         uint16_t* __restrict__ du, int64_t n, int act) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float va, vd;
    act_grad_f32(act, g[i], va, vd);
    const float d = forge::bf16_bits_to_f32(dh[i]);
    dg[i] = f32_to_bf16_bits(d * u[i] * vd);
    du[i] = f32_to_bf16_bits(d * va);
}

int64_t grad_bytes(int64_t N, int64_t I) { return forge::ceil_div(2 * N * I, 256) * 256; }

int check(const char* name, const void* rows, int64_t ldx, const int32_t* offsets, const void* Wg,
          const void* Wu, int64_t ldw, int64_t w_stride, int64_t N, int64_t E, int64_t H, int64_t I, int act) {
    FORGE_REQUIRE(N >= 0 && E >= 1 && H >= 1 && I >= 1, "%s: N=%lld E=%lld H=%lld I=%lld", name, (long long)N,
                  (long long)E, (long long)H, (long long)I);
    FORGE_REQUIRE(N <= (1 << 30) && E <= 65535 && H <= (1 << 22) && I <= (1 << 22),
                  "%s: N=%lld E=%lld H=%lld I=%lld: too large (N < 2^30, E < 2^16, H and I up to 2^22)", name,
                  (long long)N, (long long)E, (long long)H, (long long)I);
    FORGE_REQUIRE(act >= FORGE_ACT_NONE && act <= FORGE_ACT_RELU, "%s: act=%d", name, act);
    FORGE_REQUIRE(offsets && Wg && Wu && (rows || N == 0), "%s: null pointer", name);
    FORGE_REQUIRE(ldx >= H && ldw >= H && (E == 1 || w_stride >= I * ldw),
                  "%s: row pitch %lld / %lld below H=%lld or expert stride %lld below I rows", name,
                  (long long)ldx, (long long)ldw, (long long)H, (long long)w_stride);
    return FORGE_OK;
}
}  // namespace

extern "C" int forge_gated_rows(const void* rows, int64_t ldx, const int32_t* offsets, const void* Wg,
                                const void* Wu, int64_t ldw, int64_t w_stride, int64_t N, int64_t E,
                                int64_t H, int64_t I, int act, void* h, float* gate_out, float* up_out,
                                forge_stream_t stream) {
    if (int rc = check("forge_gated_rows", rows, ldx, offsets, Wg, Wu, ldw, w_stride, N, E, H, I, act)) return rc;
    if (N == 0) return FORGE_OK;
    FORGE_REQUIRE(h, "forge_gated_rows: null pointer");
    FORGE_REQUIRE((gate_out == nullptr) == (up_out == nullptr), "forge_gated_rows: gate_out and up_out go together");
    GatedArgs a{};
    a.x = (const uint16_t*)rows; a.offsets = offsets; a.wg = (const uint16_t*)Wg; a.wu = (const uint16_t*)Wu;
    a.ldx = ldx; a.ldw = ldw; a.ws = w_stride;
    a.N = (int)N; a.E = (int)E; a.H = (int)H; a.I = (int)I; a.act = act;
    a.h = (uint16_t*)h; a.g = gate_out; a.u = up_out;
    hipStream_t st = (hipStream_t)stream;
    forge::KernelTiming timing("gated_rows", st, 4.0 * N * H * I, forge::WORK_FLOPS);
    const int64_t p_tiles = forge::ceil_div(I, 32), blocks = p_tiles * forge::ragged_tiles(N, E, 64);
    FORGE_REQUIRE(blocks <= INT32_MAX, "forge_gated_rows: %lld workgroups", (long long)blocks);
    gated_any_kernel<FORWARD><<<dim3((unsigned)blocks), 256, 0, st>>>(a, (int)p_tiles);
    FORGE_LAUNCH_CHECK();
    return FORGE_OK;
}

extern "C" int64_t forge_gated_rows_backward_workspace_bytes(int64_t N, int64_t I) {
    return N > 0 && I > 0 ? 2 * grad_bytes(N, I) : 0;
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
    FORGE_REQUIRE((reinterpret_cast<uintptr_t>(ws) & 15) == 0, "%s: workspace not 16-byte aligned", name);
    uint16_t* dg = (uint16_t*)ws;
    uint16_t* du = (uint16_t*)((char*)ws + grad_bytes(N, I));
    hipStream_t st = (hipStream_t)stream;
    GatedArgs a{};
    a.x = (const uint16_t*)rows; a.offsets = offsets; a.wg = (const uint16_t*)Wg; a.wu = (const uint16_t*)Wu;
    a.ldx = ldx; a.ldw = ldw; a.ws = w_stride;
    a.N = (int)N; a.E = (int)E; a.H = (int)H; a.I = (int)I; a.act = act;
    a.dg = dg; a.du = du;
    a.dx = (uint16_t*)drows; a.dwg = (uint16_t*)dWg; a.dwu = (uint16_t*)dWu;
    const int64_t h_tiles = forge::ceil_div(H, 64), i_tiles = forge::ceil_div(I, 64);
    const int64_t blocks = h_tiles * forge::ragged_tiles(N, E, 64);
    FORGE_REQUIRE(blocks <= INT32_MAX && h_tiles * i_tiles <= INT32_MAX, "%s: too many workgroups", name);
    if (N > 0) {
        forge::KernelTiming timing("gated_grad", st, 14.0 * N * I, forge::WORK_BYTES);
        gated_grad_kernel<<<dim3((unsigned)forge::ceil_div(N * I, 256)), 256, 0, st>>>(
            (const uint16_t*)dh, g, u, dg, du, N * I, act);
        FORGE_LAUNCH_CHECK();
    }
    if (drows && N > 0) {
        forge::KernelTiming timing("gated_drows", st, 4.0 * N * H * I, forge::WORK_FLOPS);
        gated_any_kernel<DROWS><<<dim3((unsigned)blocks), 256, 0, st>>>(a, (int)h_tiles);
        FORGE_LAUNCH_CHECK();
    }
    if (dWg || dWu) {
        forge::KernelTiming timing("gated_dweights", st, 2.0 * N * H * I * ((dWg ? 1 : 0) + (dWu ? 1 : 0)), forge::WORK_FLOPS);
        // blockIdx.z picks the gate (0) or the up weights (1); one alone is passed as both
        if (!dWg) { a.dg = du; a.dwg = a.dwu; }
        gated_any_kernel<DWEIGHTS><<<dim3((unsigned)(h_tiles * i_tiles), (unsigned)E, dWg && dWu ? 2u : 1u), 256, 0, st>>>(
            a, (int)h_tiles);
        FORGE_LAUNCH_CHECK();
    }
    return FORGE_OK;
}
