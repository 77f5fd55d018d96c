// Product with packed int4 weights:  y = act(x W^T + bias) + residual,
// W[r][c] = (nibble - 8) * scale[r][c / gs].
//
// The nibbles minus 8 are integers of at most 4 bits, exact in bf16, so the matrix instruction's
// products are exact; the scale is applied to every group's f32 sum.
#include "act.h"
#include "common.h"

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
    const int64_t r_tiles = forge::ceil_div(R, 64), blocks = r_tiles * forge::ceil_div(M, 64);
    FORGE_REQUIRE(blocks <= INT32_MAX, "%s: %lld workgroups", name, (long long)blocks);
    forge::KernelTiming timing("linear_int4", st, 2.0 * M * C * R, forge::WORK_FLOPS);
    int4_any_kernel<<<dim3((unsigned)blocks), 256, 0, st>>>(a, (int)r_tiles);
    FORGE_LAUNCH_CHECK();
    return FORGE_OK;
}
