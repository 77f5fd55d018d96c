// Product with packed int4 weights:  y = act(x W^T + bias) + residual,
// W[r][c] = (nibble - 8) * scale[r][c / gs].
//
// The nibbles minus 8 are integers of at most 4 bits, exact in bf16, so the matrix instruction's
// products are exact; the scale is applied to every group's f32 sum.
#include "act.h"
#include "common.h"
#include "mfma_tile64.h"

namespace {
using forge::act_f32;
using forge::bf16_bits_to_f32;
using forge::bf16x8_t;
using forge::f32_to_bf16_bits;
using forge::f32x16_t;

struct Int4Args {
    const uint16_t* x;       // [M, C], pitch ldx
    const uint32_t* w;       // [R, words]
    const float* scale;      // [R, G]
    const uint16_t* bias;    // [R], may be null
    const uint16_t* res;     // [M, R], pitch ldr, may be null
    uint16_t* y;             // [M, R]
    int64_t ldx, ldr;
    int M, C, R, G, gs, words, act;
};

__device__ __forceinline__ void store_y(const Int4Args& a, int m, int r, float v) {
    if (a.bias) v += bf16_bits_to_f32(a.bias[r]);
    v = act_f32(a.act, v);
    if (a.res) v += bf16_bits_to_f32(a.res[(int64_t)m * a.ldr + r]);
    a.y[(int64_t)m * a.R + r] = f32_to_bf16_bits(v);
}

// Eight nibbles of a packed word as bf16 integers -8 .. 7 divided by 16, lowest first.
// v_cvt_off_f32_i4 gives a signed 4-bit integer / 16 as f32 (the top bit's flip turns offset binary into
// two's complement), exact in the upper 16 bits: 14 instructions for 8 values.  The factor 16 goes
// into the scale.
__device__ __forceinline__ bf16x8_t nibbles(uint32_t word) {
    const uint32_t a = word ^ 0x88888888u, b = a >> 4;
    uint32_t out[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t lo = __float_as_uint(__builtin_amdgcn_cvt_off_f32_i4((int)(a >> (8 * j))));
        const uint32_t hi = __float_as_uint(__builtin_amdgcn_cvt_off_f32_i4((int)(b >> (8 * j))));
        out[j] = __builtin_amdgcn_perm(hi, lo, 0x07060302u);
    }
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    const u32x4 v = {out[0], out[1], out[2], out[3]};
    return __builtin_bit_cast(bf16x8_t, v);
}
constexpr float kNibbleUnit = 16.0f;

// ---------------------------------------------------------------- few rows of x
// Bound by the packed words, which are read once: a workgroup takes 16 NT weight rows and all of
// C, its 8 wavefronts every eighth run of 128 columns, and their sums meet in LDS (in a fixed
// order).  A lane fetches 16 bytes, 32 nibbles, of one weight row, so four lanes fetch 64
// consecutive bytes of it; exchanging words between the four (two v_permlane32_swap, two
// v_permlane16_swap) gives every lane the word that the matrix instruction wants of it when each
// step takes 32 consecutive columns, and then x too is read in 64-byte runs and a step never
// crosses a group (groups are multiples of 32).  STEPS steps of 32 columns share a scale.  x comes
// from the caches: MT blocks of 16 rows; rows beyond M and columns beyond C read as zero.
template <int MT, int NT, int STEPS>
__global__ __launch_bounds__(512) void int4_few_kernel(Int4Args a) {
    using namespace forge;
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    constexpr int U = MT * NT == 1 ? 4 : MT * NT == 2 ? 2 : 1;      // runs in flight per wavefront
    constexpr int OUT = MT * NT * 256;
    __shared__ float part[8][OUT];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, kb = lane >> 4;
    const int r0 = blockIdx.x * 16 * NT, m0 = blockIdx.y * 16 * MT;
    const int rows = a.R - r0 < 16 * NT ? a.R - r0 : 16 * NT;
    const int xrows = a.M - m0 < 16 * MT ? a.M - m0 : 16 * MT;
    const __amdgpu_buffer_rsrc_t dw = descriptor(a.w + (int64_t)r0 * a.words, (uint32_t)(rows * a.words * 4));
    const __amdgpu_buffer_rsrc_t ds = descriptor(a.scale + (int64_t)r0 * a.G, (uint32_t)(rows * a.G * 4));
    const __amdgpu_buffer_rsrc_t dx = descriptor(a.x + (int64_t)m0 * a.ldx, (uint32_t)(((xrows - 1) * a.ldx + a.C) * 2));
    f32x4_t total[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) total[i][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    const int runs = (a.C + 127) / 128, full = a.words / 16;
    for (int c0 = wave; c0 < runs; c0 += 8 * U) {
        u32x4 w[U][NT], x[U][MT][4];
        float sc[U][NT][4 / STEPS];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int c = c0 + 8 * u;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const uint32_t at = (uint32_t)(((j * 16 + n) * a.words + c * 16 + kb * 4) * 4);
                if (c < full) {
                    w[u][j] = __builtin_amdgcn_raw_buffer_load_b128(dw, (int)at, 0, 0);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        w[u][j][i] = __builtin_amdgcn_raw_buffer_load_b32(
                            dw, c * 16 + kb * 4 + i < a.words ? (int)(at + 4 * i) : (int)kOutside, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < 4 / STEPS; ++i) {
                    const int k = c * 128 + i * STEPS * 32;
                    sc[u][j][i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(
                        ds, k < a.C ? ((j * 16 + n) * a.G + k / a.gs) * 4 : (int)kOutside, 0, 0));
                }
            }
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    const int k = c * 128 + d * 32 + kb * 8, m = i * 16 + n;
                    x[u][i][d] = __builtin_amdgcn_raw_buffer_load_b128(
                        dx, k < a.C && m < xrows ? (int)((m * a.ldx + k) * 2) : (int)kOutside, 0, 0);
                }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                u32x4& q = w[u][j];
                auto s = __builtin_amdgcn_permlane32_swap(q[0], q[2], false, false);
                q[0] = s[0]; q[2] = s[1];
                s = __builtin_amdgcn_permlane32_swap(q[1], q[3], false, false);
                q[1] = s[0]; q[3] = s[1];
                s = __builtin_amdgcn_permlane16_swap(q[0], q[1], false, false);
                q[0] = s[0]; q[1] = s[1];
                s = __builtin_amdgcn_permlane16_swap(q[2], q[3], false, false);
                q[2] = s[0]; q[3] = s[1];
                f32x4_t acc[MT];
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    const bf16x8_t wv = nibbles(q[d]);
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        if (d % STEPS == 0) acc[i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
                        acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, x[u][i][d]), wv,
                                                                         acc[i], 0, 0, 0);
                        if (d % STEPS == STEPS - 1)
#pragma unroll
                            for (int v = 0; v < 4; ++v)
                                total[i][j][v] = __builtin_fmaf(sc[u][j][d / STEPS], acc[i][v], total[i][j][v]);
                    }
                }
            }
    }
    // register v of a 16 x 16 block: row 4 (lane / 16) + v of x, weight row lane & 15
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int v = 0; v < 4; ++v) part[wave][((i * 16 + kb * 4 + v) * NT + j) * 16 + n] = total[i][j][v];
    __syncthreads();
    for (int o = threadIdx.x; o < OUT; o += 512) {
        const int m = m0 + o / (16 * NT), r = r0 + o % (16 * NT);
        if (m >= a.M || r >= a.R) continue;
        float v = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) v += part[i][o];
        store_y(a, m, r, v * kNibbleUnit);
    }
}

// ---------------------------------------------------------------- many rows of x
// 256 rows of x by 128 weight rows per workgroup, 64 columns a stage (mfma_tile.h), 8 wavefronts of
// 64 x 64.  x goes to LDS without registers; the packed words (two per thread and stage) are
// converted once per workgroup on their way to LDS, a stage ahead of their use.  Every group's sum
// is formed by itself and folded into the totals with its scale, one fma per output and group:
// that needs two sets of sums, which is why a wavefront has 64 x 64 outputs and not 128 x 64.
// FOLD: steps of 16 columns between folds within a stage (4: groups of 64 or more; 2: of 32).
template <int FOLD>
__global__ __launch_bounds__(512) void int4_tile_kernel(Int4Args a, int r_tiles) {
    using namespace forge;
    constexpr int kWBytes = 128 * kStage * 2;
    __shared__ __attribute__((aligned(1024))) char X0[kStageBytes], W0[kWBytes], X1[kStageBytes], W1[kWBytes];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wp = wave >> 1, wq = wave & 1;
    const int b = xcd_tile(blockIdx.x, gridDim.x);
    const int r0 = (b % r_tiles) * 128, m0 = (b / r_tiles) * kTile;
    const int rows = a.R - r0 < 128 ? a.R - r0 : 128;
    const int xrows = a.M - m0 < kTile ? a.M - m0 : kTile;
    const __amdgpu_buffer_rsrc_t dx = descriptor(a.x + (int64_t)m0 * a.ldx, (uint32_t)(((xrows - 1) * a.ldx + a.C) * 2));
    const __amdgpu_buffer_rsrc_t dw = descriptor(a.w + (int64_t)r0 * a.words, (uint32_t)(rows * a.words * 4));
    InnerLoader lx;
    lx.init(wave, lane, a.ldx, xrows, [](int t) { return t; });
    // this thread's two words of a stage: row threadIdx.x / 4, words 2 (threadIdx.x % 4) and the next
    const int wrow = threadIdx.x >> 2, wcol = (threadIdx.x & 3) * 2;
    const uint32_t wat = (uint32_t)((wrow * a.words + wcol) * 4);
    uint32_t wlds[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) wlds[i] = wrow * 128 + (((wcol + i) ^ ((wrow >> 1) & 7)) * 16);
    uint32_t word[2];
    auto fetch = [&](int s) {
        // words behind the row are a neighbour's (their x is zero) or outside the array (read as zero)
#pragma unroll
        for (int i = 0; i < 2; ++i) word[i] = __builtin_amdgcn_raw_buffer_load_b32(dw, (int)(wat + s * 32 + i * 4), 0, 0);
    };
    auto convert = [&](char* W) {
#pragma unroll
        for (int i = 0; i < 2; ++i) *reinterpret_cast<bf16x8_t*>(W + wlds[i]) = nibbles(word[i]);
    };
    InnerFragment fx, fw;
    fx.init(lane, wp * 2);
    fw.init(lane, wq * 2);
    f32x16_t total[2][2], acc[2][2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int v = 0; v < 16; ++v) total[t][n][v] = acc[t][n][v] = 0.0f;
    const float* sp[2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        const int r = r0 + (wq * 2 + n) * 32 + (lane & 31);
        sp[n] = a.scale + (int64_t)(r < a.R ? r : 0) * a.G;
    }
    int g = 0, pos = 0, end = a.gs;                             // group, columns done, where the group ends
    float sc[2] = {sp[0][0], sp[1][0]};
    auto fold = [&]() {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    total[t][n][v] = __builtin_fmaf(sc[n], acc[t][n][v], total[t][n][v]);
                    acc[t][n][v] = 0.0f;
                }
    };
    auto next_group = [&]() {
        if (++g < a.G) {
            end = a.C - end < a.gs ? a.C : end + a.gs;
            sc[0] = sp[0][g];
            sc[1] = sp[1][g];
        }
    };
    auto multiply = [&](const char* X, const char* W) {
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            bf16x8_t p[2], q[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) p[t] = fx.read(X, t, s);
#pragma unroll
            for (int t = 0; t < 2; ++t) q[t] = fw.read(W, t, s);
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int n = 0; n < 2; ++n)
                    acc[t][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(p[t], q[n], acc[t][n], 0, 0, 0);
            if (s % FOLD == FOLD - 1) {
                pos += 16 * FOLD;
                if (pos >= end && g < a.G) {
                    fold();
                    next_group();
                }
            }
        }
    };
    const int stages = (a.C + kStage - 1) / kStage;
    fetch(0);
    lx.stage(dx, X0, wave, 0, a.C);
    convert(W0);
    fetch(1);
    int s = 0;
    for (; s + 1 < stages; s += 2) {
        wait_loads();
        __syncthreads();
        lx.stage(dx, X1, wave, (s + 1) * kStage, a.C);
        convert(W1);
        fetch(s + 2);
        __builtin_amdgcn_sched_barrier(0);
        multiply(X0, W0);
        wait_loads();
        __syncthreads();
        if (s + 2 < stages) lx.stage(dx, X0, wave, (s + 2) * kStage, a.C);
        convert(W0);
        fetch(s + 3);
        __builtin_amdgcn_sched_barrier(0);
        multiply(X1, W1);
    }
    if (s < stages) {
        wait_loads();
        __syncthreads();
        multiply(X0, W0);
    }
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        const int r = r0 + (wq * 2 + n) * 32 + (lane & 31);
        if (r >= a.R) continue;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                const int m = m0 + (wp * 2 + t) * 32 + 8 * (v >> 2) + 4 * (lane >> 5) + (v & 3);
                if (m < a.M) store_y(a, m, r, total[t][n][v] * kNibbleUnit);
            }
    }
}

// Any shape, alignment and group size: 64 x 64 outputs per workgroup, four wavefronts of 32 x 32,
// 32 columns a step through LDS; a step never crosses the end of a group (its rest is zero).
__global__ __launch_bounds__(256) void int4_any_kernel(Int4Args a, int r_tiles) {
    constexpr int T = 64, K = 32, LD = K + 8;
    __shared__ uint16_t X[T][LD], W[T][LD];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = wave >> 1, wr = wave & 1;
    const int r0 = (blockIdx.x % r_tiles) * T, m0 = (blockIdx.x / r_tiles) * T;
    const int r = r0 + wr * 32 + (lane & 31);
    f32x16_t total;
#pragma unroll
    for (int v = 0; v < 16; ++v) total[v] = 0.0f;
    for (int g = 0; g < a.G; ++g) {
        const int c_end = a.C - g * a.gs < a.gs ? a.C : (g + 1) * a.gs;
        f32x16_t acc;
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[v] = 0.0f;
        for (int c0 = g * a.gs; c0 < c_end; c0 += K) {
            __syncthreads();
            for (int i = threadIdx.x; i < T * K; i += 256) {
                const int k = i % K, row = i / K, c = c0 + k;
                uint16_t xv = 0, wv = 0;
                if (c < c_end) {
                    if (m0 + row < a.M) xv = a.x[(int64_t)(m0 + row) * a.ldx + c];
                    if (r0 + row < a.R) {
                        const uint32_t word = a.w[(int64_t)(r0 + row) * a.words + c / 8];
                        wv = f32_to_bf16_bits((float)((int)((word >> (4 * (c % 8))) & 15u) - 8));
                    }
                }
                X[row][k] = xv;
                W[row][k] = wv;
            }
            __syncthreads();
#pragma unroll
            for (int s = 0; s < K; s += 16) {
                const bf16x8_t xv = *reinterpret_cast<const bf16x8_t*>(&X[wm * 32 + (lane & 31)][s + 8 * (lane >> 5)]);
                const bf16x8_t wv = *reinterpret_cast<const bf16x8_t*>(&W[wr * 32 + (lane & 31)][s + 8 * (lane >> 5)]);
                acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xv, wv, acc, 0, 0, 0);
            }
        }
        const float s = r < a.R ? a.scale[(int64_t)r * a.G + g] : 0.0f;
#pragma unroll
        for (int v = 0; v < 16; ++v) total[v] = __builtin_fmaf(s, acc[v], total[v]);
    }
    if (r >= a.R) return;
#pragma unroll
    for (int v = 0; v < 16; ++v) {
        const int m = m0 + wm * 32 + 8 * (v >> 2) + 4 * (lane >> 5) + (v & 3);
        if (m < a.M) store_y(a, m, r, total[v]);
    }
}

constexpr int64_t kFewRows = 256;    // up to here int4_few_kernel

template <int MT, int NT>
void launch_steps(const Int4Args& a, bool one_group, hipStream_t st) {
    const dim3 grid((unsigned)forge::ceil_div(a.R, 16 * NT), (unsigned)forge::ceil_div(a.M, 16 * MT));
    if (a.gs % 128 == 0 || one_group) int4_few_kernel<MT, NT, 4><<<grid, 512, 0, st>>>(a);
    else if (a.gs % 64 == 0) int4_few_kernel<MT, NT, 2><<<grid, 512, 0, st>>>(a);
    else int4_few_kernel<MT, NT, 1><<<grid, 512, 0, st>>>(a);
}
void launch_few(const Int4Args& a, bool one_group, hipStream_t st) {
    if (a.M <= 16) launch_steps<1, 1>(a, one_group, st);
    else if (a.M <= 32) launch_steps<2, 1>(a, one_group, st);
    else launch_steps<4, 1>(a, one_group, st);
}
}  // namespace

extern "C" int forge_linear_int4(const void* x, int64_t ldx, const int32_t* packed, const float* scale,
                                 int64_t gs, const void* bias, const void* residual, int64_t ldr, int64_t M,
                                 int64_t C, int64_t R, int act, void* y, forge_stream_t stream) {
    const char* name = "forge_linear_int4";
    FORGE_REQUIRE(M >= 0 && C >= 1 && R >= 1 && gs >= 1, "%s: M=%lld C=%lld R=%lld gs=%lld", name, (long long)M,
                  (long long)C, (long long)R, (long long)gs);
    FORGE_REQUIRE(M <= (1 << 30) && C <= (1 << 24) && R <= (1 << 24), "%s: M=%lld C=%lld R=%lld: too large "
                  "(M up to 2^30, C and R up to 2^24)", name, (long long)M, (long long)C, (long long)R);
    FORGE_REQUIRE(act >= FORGE_ACT_NONE && act <= FORGE_ACT_RELU, "%s: act=%d", name, act);
    if (M == 0) return FORGE_OK;
    FORGE_REQUIRE(x && packed && scale && y, "%s: null pointer", name);
    FORGE_REQUIRE(ldx >= C && (!residual || ldr >= R), "%s: row pitch %lld / %lld below C=%lld / R=%lld", name,
                  (long long)ldx, (long long)ldr, (long long)C, (long long)R);
    if (gs > C) gs = C;
    Int4Args a{(const uint16_t*)x, (const uint32_t*)packed, scale, (const uint16_t*)bias,
               (const uint16_t*)residual, (uint16_t*)y, ldx, ldr, (int)M, (int)C, (int)R,
               (int)forge::ceil_div(C, gs), (int)gs, (int)forge::ceil_div(C, 8), act};
    hipStream_t st = (hipStream_t)stream;
    forge::KernelTiming timing("linear_int4", st, 2.0 * M * C * R, forge::WORK_FLOPS);
    const bool one_group = a.G == 1;
    const bool pieces = C % 8 == 0 && ldx % 8 == 0 && ldx < (1 << 21) && (reinterpret_cast<uintptr_t>(x) & 15) == 0 &&
                        (gs % 32 == 0 || one_group);
    if (!pieces) {
        const int64_t r_tiles = forge::ceil_div(R, 64), blocks = r_tiles * forge::ceil_div(M, 64);
        FORGE_REQUIRE(blocks <= INT32_MAX, "%s: %lld workgroups", name, (long long)blocks);
        int4_any_kernel<<<dim3((unsigned)blocks), 256, 0, st>>>(a, (int)r_tiles);
    } else if (M <= kFewRows) {
        launch_few(a, one_group, st);
    } else {
        const int64_t r_tiles = forge::ceil_div(R, 128), blocks = r_tiles * forge::ceil_div(M, 256);
        FORGE_REQUIRE(blocks <= INT32_MAX, "%s: %lld workgroups", name, (long long)blocks);
        if (gs % 64 == 0 || one_group) int4_tile_kernel<4><<<dim3((unsigned)blocks), 512, 0, st>>>(a, (int)r_tiles);
        else int4_tile_kernel<2><<<dim3((unsigned)blocks), 512, 0, st>>>(a, (int)r_tiles);
    }
    FORGE_LAUNCH_CHECK();
    return FORGE_OK;
}
