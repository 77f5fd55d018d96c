// Root-mean-square norm with the residual's addition, plain and with 8-bit output.
//
//   s = x + r,  y = s * rsqrt(mean(s^2) + eps) * w,  residual out = s
//
// One pass over HBM: a row is read once into registers, summed across its lanes, and written from
// the same registers.
#include "act.h"
#include "common.h"

namespace {
using forge::bf16_bits_to_f32;
using forge::f32_to_bf16_bits;
using forge::pack_bf16;

constexpr int kGroup = 128;          // columns that share an 8-bit scale
constexpr float kFp8Max = 448.0f;    // largest e4m3fn value

struct NormArgs {
    const void* x;
    const void* res;        // may be null
    const void* w;
    void* y;                // bf16 / f32, or the e4m3 codes
    float* scale_inv;       // 8-bit output only
    void* res_out;          // null when res is
    int64_t ldx, ldr, T, C;
    float eps, inv_c;
    int w_f32;
};

// max that keeps a NaN (a run with a NaN has no scale)
__device__ __forceinline__ float nan_max(float a, float b) { return (a > b || a != a) ? a : b; }

template <typename T>
__device__ __forceinline__ float load1(const void* p, int64_t i) {
    if constexpr (sizeof(T) == 2) return bf16_bits_to_f32(((const uint16_t*)p)[i]);
    else return ((const float*)p)[i];
}
template <typename T>
__device__ __forceinline__ void store1(void* p, int64_t i, float v) {
    if constexpr (sizeof(T) == 2) ((uint16_t*)p)[i] = f32_to_bf16_bits(v);
    else ((float*)p)[i] = v;
}
template <typename T>
__device__ __forceinline__ void load8(const void* p, int64_t i, float (&v)[8]) {
    if constexpr (sizeof(T) == 2) {
        const uint4 q = *reinterpret_cast<const uint4*>((const uint16_t*)p + i);
        const uint32_t d[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[2 * j] = __uint_as_float(d[j] << 16);
            v[2 * j + 1] = __uint_as_float(d[j] & 0xFFFF0000u);
        }
    } else {
        const float4 a = *reinterpret_cast<const float4*>((const float*)p + i);
        const float4 b = *reinterpret_cast<const float4*>((const float*)p + i + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
}
template <typename T>
__device__ __forceinline__ void store8(void* p, int64_t i, const float (&v)[8]) {
    if constexpr (sizeof(T) == 2) {
        uint4 q;
        q.x = pack_bf16(v[0], v[1]); q.y = pack_bf16(v[2], v[3]);
        q.z = pack_bf16(v[4], v[5]); q.w = pack_bf16(v[6], v[7]);
        *reinterpret_cast<uint4*>((uint16_t*)p + i) = q;
    } else {
        *reinterpret_cast<float4*>((float*)p + i) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>((float*)p + i + 4) = make_float4(v[4], v[5], v[6], v[7]);
    }
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m);
    return v;
}
// e4m3fn codes of two values (v_cvt_pk_fp8_f32: nearest even; callers keep |v| <= 448 (1 + 2^-22),
// which rounds to 448)
__device__ __forceinline__ int cvt_fp8x2(float a, float b, int old, bool hi) {
    return hi ? __builtin_amdgcn_cvt_pk_fp8_f32(a, b, old, true)
              : __builtin_amdgcn_cvt_pk_fp8_f32(a, b, old, false);
}

// Quotients by one divisor, correctly rounded (P. Markstein, IBM J. Res. Dev. 34, 1990): from the correctly rounded
// reciprocal the first correction leaves a quotient within a unit of the last place, the second one the
// nearest; the residuals are exact.  A product with the reciprocal alone puts values near the middle of two codes on the
// other side, and a division per value costs 2.5 of 13 us at 4099 x 2048.  An infinite divisor gives 0, and NaN for
// an infinite value, as the division does.  (The divisors here are 2^-49 or more; quotients too small for
// exact residuals are far below the smallest code.)
struct Divisor {
    float by, inv;
    __device__ __forceinline__ explicit Divisor(float d) : by(d == INFINITY ? 0.0f : d), inv(1.0f / d) {}
    __device__ __forceinline__ float under(float v) const {
        const float q = v * inv, q1 = __builtin_fmaf(__builtin_fmaf(-by, q, v), inv, q);
        return __builtin_copysignf(__builtin_fmaf(__builtin_fmaf(-by, q1, v), inv, q1), v);      // (-0 loses its sign on the way)
    }
};

// Bound by HBM: 8192 x 7168 bf16 with a residual 96 us, 4.9 TB/s (a copy reaches 4.8); 4099 x 2048 to 8 bits 14.0 us,
// 4.2 TB/s, 1.1 us of it the quotients' corrections; one row 3.9 us, the launch and one round trip.
// LANES lanes per row, NCH runs of 8 columns per lane: lane t holds columns 8 (j LANES + t) .. + 7.
// C a multiple of 8, at most 8 LANES NCH; 16-byte aligned rows.
template <typename T, int LANES, int NCH, bool FP8>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES) void rms_norm_kernel(NormArgs a) {
    constexpr int ROWS = LANES < 256 ? 256 / LANES : 1;
    constexpr int WAVES = LANES / 64;
    __shared__ float part[WAVES];
    const int t = threadIdx.x & (LANES - 1);
    const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / LANES;
    if (ROWS > 1 && row >= a.T) return;                 // whole wavefronts leave; no barrier follows
    float s[NCH][8];
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
        const int64_t c = 8 * ((int64_t)j * LANES + t);
        if (c < a.C) {
            load8<T>(a.x, row * a.ldx + c, s[j]);
            if (a.res) {
                float r[8];
                load8<T>(a.res, row * a.ldr + c, r);
#pragma unroll
                for (int i = 0; i < 8; ++i) s[j][i] += r[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) s[j][i] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(s[j][i], s[j][i], ss);
    }
    ss = wave_sum(ss);
    if constexpr (WAVES > 1) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = ss;
        __syncthreads();
        ss = 0.0f;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) ss += part[i];
    }
    const float f = rsqrtf(__builtin_fmaf(ss, a.inv_c, a.eps));
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
        const int64_t c = 8 * ((int64_t)j * LANES + t);
        const bool in = c < a.C;
        float y[8];
        if (in) {
            if (a.res_out) store8<T>(a.res_out, row * a.C + c, s[j]);
            float w[8];
            if (a.w_f32) load8<float>(a.w, c, w); else load8<uint16_t>(a.w, c, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = s[j][i] * f * w[i];
        }
        if constexpr (!FP8) {
            if (in) store8<T>(a.y, row * a.C + c, y);
        } else {
            // a run of 128 columns = 16 neighbouring lanes
            float m = 0.0f;
            if (in) {
#pragma unroll
                for (int i = 0; i < 8; ++i) m = nan_max(m, fabsf(y[i]));
            }
#pragma unroll
            for (int k = 8; k; k >>= 1) m = nan_max(m, __shfl_xor(m, k));
            const float sc = (m < 1e-12f ? 1e-12f : m) / kFp8Max;
            if (in) {
                const Divisor d(sc);
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = d.under(y[i]);
                uint2 q;
                q.x = (uint32_t)cvt_fp8x2(y[2], y[3], cvt_fp8x2(y[0], y[1], 0, false), true);
                q.y = (uint32_t)cvt_fp8x2(y[6], y[7], cvt_fp8x2(y[4], y[5], 0, false), true);
                *reinterpret_cast<uint2*>((uint8_t*)a.y + row * a.C + c) = q;
                if ((t & 15) == 0) a.scale_inv[row * ((a.C + kGroup - 1) / kGroup) + c / kGroup] = sc;
            }
        }
    }
}

// Any C, any alignment: a workgroup per row, one column per lane and step; the row is read twice
// (the second time from the caches) because it need not fit the registers.
template <typename T, bool FP8>
__global__ __launch_bounds__(256) void rms_norm_any_kernel(NormArgs a) {
    __shared__ float part[4];
    const int64_t row = blockIdx.x;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t ox = row * a.ldx, orr = row * a.ldr;
    float ss = 0.0f;
    for (int64_t c = threadIdx.x; c < a.C; c += 256) {
        float s = load1<T>(a.x, ox + c);
        if (a.res) s += load1<T>(a.res, orr + c);
        ss = __builtin_fmaf(s, s, ss);
    }
    ss = wave_sum(ss);
    if (lane == 0) part[wave] = ss;
    __syncthreads();
    const float f = rsqrtf(__builtin_fmaf(part[0] + part[1] + part[2] + part[3], a.inv_c, a.eps));
    // a wavefront takes a run of 128 columns, two per lane
    const int64_t G = (a.C + kGroup - 1) / kGroup;
    for (int64_t g = wave; g < G; g += 4) {
        float y[2];
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int64_t c = g * kGroup + i * 64 + lane;
            y[i] = 0.0f;
            if (c < a.C) {
                float s = load1<T>(a.x, ox + c);
                if (a.res) s += load1<T>(a.res, orr + c);
                if (a.res_out) store1<T>(a.res_out, row * a.C + c, s);
                y[i] = s * f * (a.w_f32 ? load1<float>(a.w, c) : load1<uint16_t>(a.w, c));
                if constexpr (!FP8) store1<T>(a.y, row * a.C + c, y[i]);
            }
            m = nan_max(m, fabsf(y[i]));
        }
        if constexpr (FP8) {
#pragma unroll
            for (int k = 32; k; k >>= 1) m = nan_max(m, __shfl_xor(m, k));
            const float sc = (m < 1e-12f ? 1e-12f : m) / kFp8Max;
            const Divisor d(sc);
            const int q = cvt_fp8x2(d.under(y[0]), d.under(y[1]), 0, false);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int64_t c = g * kGroup + i * 64 + lane;
                if (c < a.C) ((uint8_t*)a.y)[row * a.C + c] = (uint8_t)(q >> (8 * i));
            }
            if (lane == 0) a.scale_inv[row * G + g] = sc;
        }
    }
}

template <typename T, bool FP8>
void launch(NormArgs a, bool vec, hipStream_t st) {
    // as many rows at a time as a launch can have threads for
    const int width = !vec ? 0 : a.C <= 64 * 8 * 4 ? 64 : a.C <= 256 * 8 * 4 ? 256 : a.C <= 1024 * 8 * 2 ? 1024 : 0;
    const int64_t T0 = a.T, most = width == 64 ? forge::max_workgroups(256) * 4 : forge::max_workgroups(width == 1024 ? 1024 : 256);
    for (int64_t done = 0; done < T0; done += a.T) {
        a.T = T0 - done < most ? T0 - done : most;
        const dim3 grid((unsigned)(width == 64 ? forge::ceil_div(a.T, 4) : a.T));
        if (width == 64) rms_norm_kernel<T, 64, 4, FP8><<<grid, 256, 0, st>>>(a);
        else if (width == 256) rms_norm_kernel<T, 256, 4, FP8><<<grid, 256, 0, st>>>(a);
        else if (width == 1024) rms_norm_kernel<T, 1024, 2, FP8><<<grid, 1024, 0, st>>>(a);
        else rms_norm_any_kernel<T, FP8><<<grid, 256, 0, st>>>(a);
        a.x = (const T*)a.x + a.T * a.ldx;
        if (a.res) {
            a.res = (const T*)a.res + a.T * a.ldr;
            a.res_out = (T*)a.res_out + a.T * a.C;
        }
        a.y = (char*)a.y + a.T * a.C * (FP8 ? 1 : sizeof(T));
        if (FP8) a.scale_inv += a.T * forge::ceil_div(a.C, kGroup);
    }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int rms_norm(const char* name, const void* x, int dtype, int64_t ldx, const void* residual, int64_t ldr,
             const void* weight, int w_dtype, int64_t T, int64_t C, float eps, void* y, float* scale_inv,
             void* residual_out, bool fp8, forge_stream_t stream) {
    FORGE_REQUIRE(dtype == FORGE_F32 || dtype == FORGE_BF16, "%s: dtype=%d", name, dtype);
    FORGE_REQUIRE(w_dtype == FORGE_F32 || w_dtype == FORGE_BF16, "%s: w_dtype=%d", name, w_dtype);
    FORGE_REQUIRE(T >= 0 && C >= 1, "%s: T=%lld C=%lld", name, (long long)T, (long long)C);
    FORGE_REQUIRE(T <= INT32_MAX && C <= INT32_MAX, "%s: T=%lld, C=%lld: more than 2^31 - 1", name,
                  (long long)T, (long long)C);
    FORGE_REQUIRE(eps >= 0.0f, "%s: eps=%g", name, eps);
    if (T == 0) return FORGE_OK;
    FORGE_REQUIRE(x && weight && y && (!fp8 || scale_inv), "%s: null pointer", name);
    FORGE_REQUIRE((residual == nullptr) == (residual_out == nullptr),
                  "%s: residual and residual_out go together", name);
    FORGE_REQUIRE(ldx >= C && (!residual || ldr >= C), "%s: row pitch %lld / %lld below C=%lld", name,
                  (long long)ldx, (long long)ldr, (long long)C);
    const int64_t size = dtype == FORGE_BF16 ? 2 : 4;
    const bool vec = C % 8 == 0 && ldx % 8 == 0 && (!residual || ldr % 8 == 0) && aligned16(x) &&
                     aligned16(weight) && aligned16(y) && aligned16(residual) && aligned16(residual_out);
    NormArgs a{x, residual, weight, y, scale_inv, residual_out, ldx, ldr, T, C, eps, 1.0f / (float)C,
               w_dtype == FORGE_F32};
    hipStream_t st = (hipStream_t)stream;
    const double bytes = (double)T * C * (size * (residual ? 3 : 1) + (fp8 ? 1 : size));
    forge::KernelTiming timing(name + 6, st, bytes, forge::WORK_BYTES);
    if (dtype == FORGE_BF16) {
        if (fp8) launch<uint16_t, true>(a, vec, st); else launch<uint16_t, false>(a, vec, st);
    } else {
        if (fp8) launch<float, true>(a, vec, st); else launch<float, false>(a, vec, st);
    }
    FORGE_LAUNCH_CHECK();
    return FORGE_OK;
}
}  // namespace

extern "C" int forge_rms_norm(const void* x, int dtype, int64_t ldx, const void* residual, int64_t ldr,
                              const void* weight, int w_dtype, int64_t T, int64_t C, float eps, void* y,
                              void* residual_out, forge_stream_t stream) {
    return rms_norm("forge_rms_norm", x, dtype, ldx, residual, ldr, weight, w_dtype, T, C, eps, y, nullptr,
                    residual_out, false, stream);
}

extern "C" int forge_rms_norm_fp8(const void* x, int dtype, int64_t ldx, const void* residual, int64_t ldr,
                                  const void* weight, int w_dtype, int64_t T, int64_t C, float eps,
                                  uint8_t* codes, float* scale_inv, void* residual_out,
                                  forge_stream_t stream) {
    return rms_norm("forge_rms_norm_fp8", x, dtype, ldx, residual, ldr, weight, w_dtype, T, C, eps, codes,
                    scale_inv, residual_out, true, stream);
}
