// Product with packed int4 weights:  y = act(x W^T + bias) + residual,
// W[r][c] = (code - zero[r][c / gs]) * scale[r][c / gs].
//
// A nibble is code - zero + 8 modulo 16.  Without zero points (they are all 8, symmetric grids) it is the code, and
// nibble - 8 is a signed 4-bit integer; with them code - zero takes five bits, so the code is formed
// again from the nibble and the zero point (ZERO).  Either is exact in bf16, so the matrix instruction's
// products are exact; the scale is applied to every group's f32 sum.
#include "act.h"
#include "common.h"
#include "mfma_tile.h"

#include <type_traits>

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
    const int32_t* zero;     // [R, G], null without zero points
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

// the same for 8 columns (R, ldr and the pointers allow 16-byte accesses), whose bias and residual the caller has
// loaded beforehand
__device__ __forceinline__ uint4 load_bias8(const Int4Args& a, int r) {
    return a.bias ? *reinterpret_cast<const uint4*>(a.bias + r) : make_uint4(0, 0, 0, 0);
}
__device__ __forceinline__ uint4 load_residual8(const Int4Args& a, int m, int r) {
    return a.res ? *reinterpret_cast<const uint4*>(a.res + (int64_t)m * a.ldr + r) : make_uint4(0, 0, 0, 0);
}
__device__ __forceinline__ void store_y8(const Int4Args& a, int m, int r, float (&v)[8], const uint4& bias, const uint4& residual) {
    const uint32_t b[4] = {bias.x, bias.y, bias.z, bias.w}, e[4] = {residual.x, residual.y, residual.z, residual.w};
    uint32_t y[4];
    if (a.bias) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] += __uint_as_float(k & 1 ? b[k / 2] & 0xFFFF0000u : b[k / 2] << 16);
    }
    forge::act_all(a.act, v);
    if (a.res) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] += __uint_as_float(k & 1 ? e[k / 2] & 0xFFFF0000u : e[k / 2] << 16);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) y[k] = forge::pack_bf16(v[2 * k], v[2 * k + 1]);
    *reinterpret_cast<uint4*>(a.y + (int64_t)m * a.R + r) = make_uint4(y[0], y[1], y[2], y[3]);
}

// The low nibble of byte B as a signed 4-bit integer / 16, f32: the instruction's operand is the byte
// itself (left to itself the compiler shifts every nibble down first)
template <int B>
__device__ __forceinline__ uint32_t nibble_of_byte(uint32_t v) {
    uint32_t r;
    if constexpr (B == 0) asm("v_cvt_off_f32_i4_sdwa %0, %1 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_0" : "=v"(r) : "v"(v));
    else if constexpr (B == 1) asm("v_cvt_off_f32_i4_sdwa %0, %1 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1" : "=v"(r) : "v"(v));
    else if constexpr (B == 2) asm("v_cvt_off_f32_i4_sdwa %0, %1 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2" : "=v"(r) : "v"(v));
    else asm("v_cvt_off_f32_i4_sdwa %0, %1 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3" : "=v"(r) : "v"(v));
    return r;
}
// Eight nibbles of a packed word as bf16 integers -8 .. 7 divided by 16, lowest first.
// v_cvt_off_f32_i4 gives a signed 4-bit integer / 16 as f32 (the top bit's flip turns offset binary into
// two's complement), exact in the upper 16 bits: 14 instructions for 8 values.  The factor 16 goes
// into the scale.
__device__ __forceinline__ bf16x8_t nibbles(uint32_t word) {
    const uint32_t a = word ^ 0x88888888u, b = a >> 4;
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    const u32x4 v = {__builtin_amdgcn_perm(nibble_of_byte<0>(b), nibble_of_byte<0>(a), 0x07060302u),
                     __builtin_amdgcn_perm(nibble_of_byte<1>(b), nibble_of_byte<1>(a), 0x07060302u),
                     __builtin_amdgcn_perm(nibble_of_byte<2>(b), nibble_of_byte<2>(a), 0x07060302u),
                     __builtin_amdgcn_perm(nibble_of_byte<3>(b), nibble_of_byte<3>(a), 0x07060302u)};
    return __builtin_bit_cast(bf16x8_t, v);
}
constexpr float kNibbleUnit = 16.0f;

// A group's zero point as nibbles() takes it: in all eight nibbles of a word, and (8 - zero) / 16
struct Zero {
    uint32_t add;
    float off;
};
__device__ __forceinline__ Zero zero_of(uint32_t z) {
    return {(z & 15u) * 0x11111111u, __builtin_fmaf(-0.0625f, (float)(int)z, 0.5f)};
}
// The eight values code - zero of a word as bf16, divided by 16 like those above.  nibble + zero modulo 16 is code - 8
// as a signed 4-bit integer (added in the low three bits of every nibble, the top bit by exclusive or: nothing
// carries into a neighbour); (code - 8) / 16 + (8 - zero) / 16 is exact, in the upper 16 bits too (zero within
// -240 .. 255).  26 instructions for 8 values: one row, 2048 -> 7168, 5.8 us against 4.9; 8192 rows 515 / 446.
__device__ __forceinline__ bf16x8_t nibbles(uint32_t word, const Zero& z) {
    const uint32_t a = ((word & 0x77777777u) + (z.add & 0x77777777u)) ^ ((word ^ z.add) & 0x88888888u), b = a >> 4;
    auto value = [&](uint32_t v) { return __float_as_uint(__uint_as_float(v) + z.off); };
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    const u32x4 v = {__builtin_amdgcn_perm(value(nibble_of_byte<0>(b)), value(nibble_of_byte<0>(a)), 0x07060302u),
                     __builtin_amdgcn_perm(value(nibble_of_byte<1>(b)), value(nibble_of_byte<1>(a)), 0x07060302u),
                     __builtin_amdgcn_perm(value(nibble_of_byte<2>(b)), value(nibble_of_byte<2>(a)), 0x07060302u),
                     __builtin_amdgcn_perm(value(nibble_of_byte<3>(b)), value(nibble_of_byte<3>(a)), 0x07060302u)};
    return __builtin_bit_cast(bf16x8_t, v);
}
template <bool ZERO>
__device__ __forceinline__ bf16x8_t weights(uint32_t word, const Zero& z) {
    if constexpr (ZERO) return nibbles(word, z);
    else return nibbles(word);
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t zero_descriptor(const Int4Args& a, int r0, int rows) {
    return forge::descriptor(a.zero + (int64_t)r0 * a.G, (uint32_t)(rows * a.G * 4));
}

// ---------------------------------------------------------------- few rows of x
// Bound by the packed words, which are read once: a workgroup takes 16 weight rows, its 8 wavefronts every
// eighth run of 128 columns, and their sums meet in LDS (in a fixed order; fewer wavefronts per row and
// more rows per workgroup were slower at every size, 47 against 34 us then at 7168 -> 18432).  A lane fetches
// 16 bytes, 32 nibbles, of one weight row, so four lanes fetch 64 consecutive bytes of it; exchanging
// words between the four (two v_permlane32_swap, two v_permlane16_swap) gives every lane the word that
// the matrix instruction wants of it when each step takes 32 consecutive columns, and then x too is read
// in 64-byte runs and a step never crosses a group (groups are multiples of 32).  STEPS steps of 32 columns share a
// scale.  The up to 16 rows of x come from the caches; rows beyond M and columns beyond C read as zero.
template <int STEPS, bool ZERO>
__global__ __launch_bounds__(512) void int4_few_kernel(Int4Args a) {
    using namespace forge;
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    __shared__ float part[8][256];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, kb = lane >> 4;
    const int r0 = blockIdx.x * 16, rows = min(a.R - r0, 16);
    const __amdgpu_buffer_rsrc_t dw = descriptor(a.w + (int64_t)r0 * a.words, (uint32_t)(rows * a.words * 4));
    const __amdgpu_buffer_rsrc_t ds = descriptor(a.scale + (int64_t)r0 * a.G, (uint32_t)(rows * a.G * 4));
    const __amdgpu_buffer_rsrc_t dx = descriptor(a.x, (uint32_t)(((a.M - 1) * a.ldx + a.C) * 2));
    __amdgpu_buffer_rsrc_t dz;
    if constexpr (ZERO) dz = zero_descriptor(a, r0, rows);
    f32x4_t total = {0.0f, 0.0f, 0.0f, 0.0f};
    const int runs = (a.C + 127) / 128;
    // One run at a time: the other wavefronts' are on their way meanwhile (two or four of each asked for at once
    // keep wavefronts off the CU: 2048 -> 7168, 1 row 7.8 us with one, 9.5 with four; 7168 -> 18432 28.8 / 31.5)
    for (int c = wave; c < runs; c += 8) {
        u32x4 x[4];
        float sc[4 / STEPS];
        Zero z[4 / STEPS] = {};
        // (words behind the row are a neighbour's, their x is zero, or outside the array)
        u32x4 q = __builtin_amdgcn_raw_buffer_load_b128(dw, (n * a.words + c * 16 + kb * 4) * 4, 0, 0);
#pragma unroll
        for (int i = 0; i < 4 / STEPS; ++i) {
            const int k = c * 128 + i * STEPS * 32;
            const int at = k < a.C ? (n * a.G + k / a.gs) * 4 : (int)kOutside;
            sc[i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(ds, at, 0, 0));
            if constexpr (ZERO) z[i] = zero_of(__builtin_amdgcn_raw_buffer_load_b32(dz, at, 0, 0));
        }
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            const int k = c * 128 + d * 32 + kb * 8;
            x[d] = __builtin_amdgcn_raw_buffer_load_b128(
                dx, k < a.C && n < a.M ? (int)((n * a.ldx + k) * 2) : (int)kOutside, 0, 0);
        }
        auto s = __builtin_amdgcn_permlane32_swap(q[0], q[2], false, false);
        q[0] = s[0]; q[2] = s[1];
        s = __builtin_amdgcn_permlane32_swap(q[1], q[3], false, false);
        q[1] = s[0]; q[3] = s[1];
        s = __builtin_amdgcn_permlane16_swap(q[0], q[1], false, false);
        q[0] = s[0]; q[1] = s[1];
        s = __builtin_amdgcn_permlane16_swap(q[2], q[3], false, false);
        q[2] = s[0]; q[3] = s[1];
        f32x4_t acc;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            if (d % STEPS == 0) acc = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, x[d]), weights<ZERO>(q[d], z[d / STEPS]), acc, 0, 0, 0);
            if (d % STEPS == STEPS - 1)
#pragma unroll
                for (int v = 0; v < 4; ++v) total[v] = __builtin_fmaf(sc[d / STEPS], acc[v], total[v]);
        }
    }
    // register v: row 4 (lane / 16) + v of x, weight row lane & 15
#pragma unroll
    for (int v = 0; v < 4; ++v) part[wave][(kb * 4 + v) * 16 + n] = total[v];
    __syncthreads();
    if (threadIdx.x >= 256) return;
    const int m = threadIdx.x / 16, r = r0 + threadIdx.x % 16;
    if (m >= a.M || r >= a.R) return;
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) v += part[w][threadIdx.x];
    store_y(a, m, r, v * kNibbleUnit);
}

// ---------------------------------------------------------------- many rows of x
// 128 rows of x by 256 weight rows per workgroup, 64 columns a stage (mfma_tile.h).  A wavefront takes all of
// the rows of x by 32 weight rows: a 32 x 16 fragment of W is one word per lane, converted by the only
// wavefront that multiplies by it, a step ahead.  8192 rows, 7168 -> 4096: 450 us, 1070 TFLOP/s
// (469 with bias, activation and residual; 515 with zero points), the clock at 1.6 to 1.7 GHz (2.1 and more where power
// allows), the matrix pipe busy for half of the cycles and the vector ALU for half, so what counts is the work itself: 64 x 64 outputs per wavefront halve the reads of x from LDS
// but convert every word twice (585 us against 490 at that time).  Converted once, into LDS, words cost 16 KB of
// writes and 64 KB of reads a stage.
// Every group's sum is formed by itself and folded into the totals with its scale, one fma per output and
// group: that needs two sets of sums, which is why a wavefront has 64 x 64 outputs' worth and not twice that.
// x and the packed words go to LDS without registers, four stages ahead, the words in runs of 64 bytes
// (two stages: a lane's own 16 bytes of its weight row, straight into registers, are a request each, and
// 16 such loads a stage keep the address unit busy longer than the matrix pipe).
// Where groups end is fixed at compile time: 128 columns (two stages) hold FOLDS folds (1: groups of
// 128 k or a single one; 2: of 64 k; 4: of 32 k).  The first product of a group starts from the
// constant zero.
template <int FOLDS, bool ZERO>
__global__ __launch_bounds__(512) void int4_tile_kernel(Int4Args a, int r_tiles, int m_tiles, bool vec) {
    using namespace forge;
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    constexpr int kRows = 128, kXBytes = kRows * kStage * 2;
    // (the epilogue takes half of the tile's 128 KB in f32 at a time)
    __shared__ __attribute__((aligned(1024))) char X0[kXBytes], X1[kXBytes], X2[kXBytes], X3[kXBytes], W0[256 * 64], W1[256 * 64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tile = xcd_tile(blockIdx.x, r_tiles * m_tiles);
    if (tile >= r_tiles * m_tiles) return;
    // runs of 8 tiles of x by all weight tiles
    const int run = tile / (8 * r_tiles), in_run = tile - run * 8 * r_tiles, wide = min(m_tiles - run * 8, 8);
    const int r0 = in_run / wide * 256, m0 = (run * 8 + in_run % wide) * kRows;
    const int rows = min(a.R - r0, 256), xrows = min(a.M - m0, kRows);
    const __amdgpu_buffer_rsrc_t dx = descriptor(a.x + (int64_t)m0 * a.ldx, (uint32_t)(((xrows - 1) * a.ldx + a.C) * 2));
    const __amdgpu_buffer_rsrc_t dw = descriptor(a.w + (int64_t)r0 * a.words, (uint32_t)(rows * a.words * 4));
    const __amdgpu_buffer_rsrc_t ds = descriptor(a.scale + (int64_t)r0 * a.G, (uint32_t)(rows * a.G * 4));
    __amdgpu_buffer_rsrc_t dz;
    if constexpr (ZERO) dz = zero_descriptor(a, r0, rows);
    InnerLoader<2> lx;
    lx.init(lane, a.ldx, wave * 16);
    InnerFragment fx;
    fx.init(lane, 0);

    const uint32_t sat = (uint32_t)((wave * 32 + (lane & 31)) * a.G * 4);
    // Words of two stages: row r at 64 r, its 16-byte piece c (2 (stage % 2) + lane / 32 of the reader) at
    // c ^ (r / 4 % 4).  What lies behind the row is a neighbour's (its x is zero) or outside the array: the
    // range check is per word, so a load across the array's end still gets the words inside.
    const uint32_t wat = (uint32_t)((wave * 32 + lane / 4) * a.words * 4 + (((lane & 3) ^ ((lane >> 4) & 3)) * 16));
    auto load_words = [&](char* W, int pair) {
#pragma unroll
        for (int j = 0; j < 2; ++j) load_to_lds(dw, W + (wave * 2 + j) * 1024, wat + (uint32_t)(j * 64 * a.words) + pair * 64);
    };
    const uint32_t wfrom = (uint32_t)((wave * 32 + (lane & 31)) * 64);
    auto read_words = [&](u32x4& w, const char* W, int odd) {
        w = *reinterpret_cast<const u32x4*>(W + wfrom + (((odd * 2 + (lane >> 5)) ^ ((lane >> 2) & 3)) * 16));
    };
    // words 0 .. 3 | 4 .. 7 of the two lanes to 0 2 4 6 | 1 3 5 7: word of step s is then 2 s + lane / 32
    auto spread = [&](u32x4& w) {
        auto p = __builtin_amdgcn_permlane32_swap(w[0], w[1], false, false);
        auto q = __builtin_amdgcn_permlane32_swap(w[2], w[3], false, false);
        w[0] = p[0]; w[2] = p[1];
        w[1] = q[0]; w[3] = q[1];
    };

    f32x16_t total[4], acc[4];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int v = 0; v < 16; ++v) total[t][v] = 0.0f;
    // The scales of the four stages of a turn's folds, each asked for when the turn before has used its
    // place: loads come back in order, so a wait for a young one is a wait for all x and words before it
    // (asked for two stages ahead they cost half of the kernel's time).
    constexpr int kFolds = 2 * FOLDS;
    uint32_t sc[kFolds];
    int g = 0, k_next = 0, k_end = a.gs;                        // of the group whose scales are asked for next
    auto scales = [&](int i) {
        sc[i] = __builtin_amdgcn_raw_buffer_load_b32(ds, (int)(sat + g * 4), 0, 0);
        k_next += 128 / FOLDS;
        if (k_next >= k_end && g + 1 < a.G) {                   // (the last group's again behind C)
            ++g;
            k_end += a.gs;
        }
    };
    // Zero points the same way, but a group's is wanted before its first conversion, which is before the
    // group in front of it is folded: they are asked for one group further ahead, and the place of
    // fold i + 1 is free when fold i is made.
    constexpr int kAsked = ZERO ? 2 : 1;                        // loads per fold
    uint32_t zr[kFolds];
    Zero zero = {};
    int gz = 0, kz_next = 0, kz_end = a.gs;
    auto zeros = [&](uint32_t& to) {
        to = __builtin_amdgcn_raw_buffer_load_b32(dz, (int)(sat + gz * 4), 0, 0);
        kz_next += 128 / FOLDS;
        if (kz_next >= kz_end && gz + 1 < a.G) {
            ++gz;
            kz_end += a.gs;
        }
    };
    auto group = [&](int i) {                                   // the words that follow belong to fold i
        if constexpr (ZERO) zero = zero_of(zr[i]);
    };
    auto fold = [&](int i) {
        const float scale = __uint_as_float(sc[i]);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int v = 0; v < 16; ++v) total[t][v] = __builtin_fmaf(scale, acc[t][v], total[t][v]);
            // here and now: put off, several groups' sums would be alive at once, 64 registers each
            asm volatile("" : "+v"(total[t]));
        }
        scales(i);
        if constexpr (ZERO) zeros(zr[(i + 1) % kFolds]);
    };
    struct Step {
        bf16x8_t p[4], q;
    };
    auto prepare = [&](Step& f, const char* X, int s, const u32x4& w) {
#pragma unroll
        for (int t = 0; t < 4; ++t) f.p[t] = fx.read(X, t, s);
        f.q = weights<ZERO>(w[s], zero);
    };
    auto multiply = [&](auto first, const Step& f) {
        const f32x16_t zero = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < 4; ++t)
            acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f.p[t], f.q, decltype(first)::value ? zero : acc[t], 0, 0, 0);
        // a step's matrix instructions among the next step's reads (and conversions, as the compiler likes)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    Step f, h;
    // Stage s, the I-th of its turn; the next one's x in Xn.  w: its words (spread), wn: the next stage's;
    // W: this pair of stages' words, Wn: the next pair's
    auto one_stage = [&](auto i, int s, char* X, const char* Xn, char* W, const char* Wn, u32x4& w, u32x4& wn) {
        constexpr int I = decltype(i)::value;
        constexpr bool kFirst = I % 2 == 0 || FOLDS > 1, kLast = I % 2 == 1 || FOLDS > 1;
        prepare(h, X, 1, w);
        multiply(std::integral_constant<bool, kFirst>{}, f);
        if (FOLDS == 4) group(2 * I + 1);
        prepare(f, X, 2, w);
        multiply(std::false_type{}, h);
        if (FOLDS == 4) fold(2 * I);
        prepare(h, X, 3, w);
        multiply(std::integral_constant<bool, FOLDS == 4>{}, f);
        // The next stage's x (and words, if a pair begins) have arrived once no more loads are on their way
        // than were issued behind them: x of two stages, one pair's words, and the scales (and zero points) of
        // three stages (FOLDS 1: of every other).
        constexpr int kScales = FOLDS == 1 ? (I % 2 == 0 ? 2 : 1) : FOLDS == 2 ? 3 : 6;
        wait_loads_barrier<2 * 2 + 2 + kAsked * kScales>();
        lx.stage(dx, X, wave, a.ldx, (s + 4) * kStage, a.C);
        __builtin_amdgcn_sched_barrier(0);
        if (I % 2 == 0) {
            load_words(W, s / 2 + 2);                           // everybody has this pair's in registers
            __builtin_amdgcn_sched_barrier(0);
        } else {
            read_words(wn, Wn, 0);
            read_words(w, Wn, 1);
        }
        spread(wn);
        if (kLast) group(FOLDS == 1 ? (I + 1) / 2 % 2 : (I + 1) * (FOLDS / 2) % kFolds);
        prepare(f, Xn, 0, wn);
        multiply(std::false_type{}, h);
        if (kLast) fold(FOLDS == 1 ? I / 2 : FOLDS == 2 ? I : 2 * I + 1);
    };
    u32x4 w0, w1;                                               // words of even and odd stages
    uint32_t first_zero;
    if constexpr (ZERO) zeros(first_zero);
    __builtin_amdgcn_sched_barrier(0);
    // in the loop's own order
    lx.stage(dx, X0, wave, a.ldx, 0, a.C);
    __builtin_amdgcn_sched_barrier(0);
    load_words(W0, 0);
    __builtin_amdgcn_sched_barrier(0);
    lx.stage(dx, X1, wave, a.ldx, kStage, a.C);
    lx.stage(dx, X2, wave, a.ldx, 2 * kStage, a.C);
    __builtin_amdgcn_sched_barrier(0);
    load_words(W1, 1);
    __builtin_amdgcn_sched_barrier(0);
    lx.stage(dx, X3, wave, a.ldx, 3 * kStage, a.C);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < kFolds; ++i) {
        scales(i);
        if constexpr (ZERO) zeros(zr[(i + 1) % kFolds]);
    }
    wait_loads_barrier<8 + kAsked * kFolds>();
    read_words(w0, W0, 0);
    read_words(w1, W0, 1);
    spread(w0);
    if constexpr (ZERO) zero = zero_of(first_zero);
    prepare(f, X0, 0, w0);
    // (columns behind C are zeros of x times a neighbour's words)
    const int stages = (a.C + 2 * kStage - 1) / (2 * kStage) * 2;
    int s = 0;
    for (; s + 4 <= stages; s += 4) {
        one_stage(std::integral_constant<int, 0>{}, s, X0, X1, W0, W1, w0, w1);
        one_stage(std::integral_constant<int, 1>{}, s + 1, X1, X2, W0, W1, w1, w0);
        one_stage(std::integral_constant<int, 2>{}, s + 2, X2, X3, W1, W0, w0, w1);
        one_stage(std::integral_constant<int, 3>{}, s + 3, X3, X0, W1, W0, w1, w0);
    }
    if (s < stages) {
        one_stage(std::integral_constant<int, 0>{}, s, X0, X1, W0, W1, w0, w1);
        one_stage(std::integral_constant<int, 1>{}, s + 1, X1, X2, W0, W1, w1, w0);
    }
    wait_loads<0>();
    __syncthreads();
    // The tile goes through LDS as f32, 64 rows of x at a time, so that bias,
    // residual and y are read and written in runs of 8 columns.  16 rows of 1 KB a buffer.
    // Register v of a tile: row 8 (v / 4) + 4 (lane / 32) + v % 4 of x, weight row lane & 31.
    auto quarter = [&](int i) { return reinterpret_cast<float*>(i == 0 ? X0 : i == 1 ? X1 : i == 2 ? X2 : X3); };
    // 32 threads a row, 16 rows at a time; what is added is asked for before the tile is in LDS
    const int c = (threadIdx.x & 31) * 8, r = r0 + c;
    const bool pieces = vec && r < a.R;
    const uint4 none = make_uint4(0, 0, 0, 0), bias = pieces ? load_bias8(a, r) : none;
#pragma unroll
    for (int pass = 0; pass < 2; ++pass) {
        uint4 residual[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int m = m0 + pass * 64 + i * 16 + (threadIdx.x >> 5);
            residual[i] = pieces && m < a.M ? load_residual8(a, m, r) : none;
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int v = 0; v < 16; ++v)
                quarter(t * 2 + (v >> 3))[(8 * ((v >> 2) & 1) + 4 * (lane >> 5) + (v & 3)) * 256 + wave * 32 + (lane & 31)] =
                    total[pass * 2 + t][v] * kNibbleUnit;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int m = m0 + pass * 64 + i * 16 + (threadIdx.x >> 5);
            if (m >= a.M || r >= a.R) continue;
            const float* from = quarter(i) + (threadIdx.x >> 5) * 256 + c;
            if (vec) {
                float v[8];
                *reinterpret_cast<f32x4_t*>(v) = *reinterpret_cast<const f32x4_t*>(from);
                *reinterpret_cast<f32x4_t*>(v + 4) = *reinterpret_cast<const f32x4_t*>(from + 4);
                store_y8(a, m, r, v, bias, residual[i]);
            } else {
                for (int k = 0; k < 8 && r + k < a.R; ++k) store_y(a, m, r + k, from[k]);
            }
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------- in between
// Too many rows of x for the kernel above to read them from the caches for every 16 weight rows, too
// few for 128 x 256 tiles to fill the GPU: 32 PT rows of x by 64 weight rows per workgroup, and each of its 8
// wavefronts forms all of that tile over every eighth 128 columns (a pair of stages), on LDS buffers of
// its own, without a barrier; their sums meet in LDS in a fixed order.  The wavefront's inner loop is
// that of the tiles: x a stage ahead, words a pair ahead, fragments a step ahead.
template <int PT, int FOLDS, bool ZERO>
__global__ __launch_bounds__(512) void int4_split_kernel(Int4Args a, int r_tiles, int m_tiles, bool vec) {
    using namespace forge;
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    constexpr int kRows = 32 * PT, kXBytes = kRows * 128;
    __shared__ __attribute__((aligned(1024))) char XA[8 * kXBytes], XB[8 * kXBytes], W[8 * 4096];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tile = xcd_tile(blockIdx.x, r_tiles * m_tiles);
    if (tile >= r_tiles * m_tiles) return;
    const int r0 = tile / m_tiles * 64, m0 = tile % m_tiles * kRows;
    const int rows = min(a.R - r0, 64), xrows = min(a.M - m0, kRows);
    const __amdgpu_buffer_rsrc_t dx = descriptor(a.x + (int64_t)m0 * a.ldx, (uint32_t)(((xrows - 1) * a.ldx + a.C) * 2));
    const __amdgpu_buffer_rsrc_t dw = descriptor(a.w + (int64_t)r0 * a.words, (uint32_t)(rows * a.words * 4));
    const __amdgpu_buffer_rsrc_t ds = descriptor(a.scale + (int64_t)r0 * a.G, (uint32_t)(rows * a.G * 4));
    __amdgpu_buffer_rsrc_t dz;
    if constexpr (ZERO) dz = zero_descriptor(a, r0, rows);
    InnerLoader<4 * PT> lx;                                     // as wavefront 0 of a tile of its own
    lx.init(lane, a.ldx, 0);
    InnerFragment fx;
    fx.init(lane, 0);
    // words of a pair of stages: row r at 64 r, its piece c at c ^ (r / 4 % 4)
    const uint32_t wat = (uint32_t)((lane / 4) * a.words * 4 + (((lane & 3) ^ ((lane >> 4) & 3)) * 16));
    const uint32_t wfrom = (uint32_t)(wave * 4096 + (lane & 31) * 64);
    char *const xa = XA + wave * kXBytes, *const xb = XB + wave * kXBytes;
    auto load_x = [&](char* X, int k) { lx.stage(dx, X, 0, a.ldx, k, a.C); };
    auto load_words = [&](int pair) {
#pragma unroll
        for (int j = 0; j < 4; ++j) load_to_lds(dw, W + wave * 4096 + j * 1024, wat + (uint32_t)(j * 64 * a.words) + pair * 64);
    };
    auto read_words = [&](u32x4 (&w)[2], int odd) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            w[n] = *reinterpret_cast<const u32x4*>(W + wfrom + n * 2048 + (((odd * 2 + (lane >> 5)) ^ ((lane >> 2) & 3)) * 16));
        }
    };
    auto spread = [&](u32x4 (&w)[2]) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            auto p = __builtin_amdgcn_permlane32_swap(w[n][0], w[n][1], false, false);
            auto q = __builtin_amdgcn_permlane32_swap(w[n][2], w[n][3], false, false);
            w[n][0] = p[0]; w[n][2] = p[1];
            w[n][1] = q[0]; w[n][3] = q[1];
        }
    };
    f32x16_t total[PT][2], acc[PT][2];
#pragma unroll
    for (int t = 0; t < PT; ++t)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int v = 0; v < 16; ++v) total[t][n][v] = 0.0f;
    const uint32_t sat = (uint32_t)(lane * a.G * 4);
    auto scales = [&](__amdgpu_buffer_rsrc_t d, uint32_t (&sc)[FOLDS], int pair) {
        int g = pair * 128 / a.gs, into = pair * 128 - g * a.gs;
#pragma unroll
        for (int i = 0; i < FOLDS; ++i) {
            sc[i] = __builtin_amdgcn_raw_buffer_load_b32(d, (int)(sat + min(g, a.G - 1) * 4), 0, 0);
            into += 128 / FOLDS;
            if (into >= a.gs) {
                into -= a.gs;
                ++g;
            }
        }
    };
    // the zero points of the words that follow, from what was loaded like the scales
    Zero zero[2] = {};
    auto group = [&](uint32_t z) {
        const auto both = __builtin_amdgcn_permlane32_swap(z, z, false, false);
        zero[0] = zero_of(both[0]);
        zero[1] = zero_of(both[1]);
    };
    auto fold = [&](uint32_t s) {
        const auto both = __builtin_amdgcn_permlane32_swap(s, s, false, false);
        const float s2[2] = {__uint_as_float(both[0]), __uint_as_float(both[1])};
#pragma unroll
        for (int t = 0; t < PT; ++t)
#pragma unroll
            for (int n = 0; n < 2; ++n) {
#pragma unroll
                for (int v = 0; v < 16; ++v) total[t][n][v] = __builtin_fmaf(s2[n], acc[t][n][v], total[t][n][v]);
                asm volatile("" : "+v"(total[t][n]));           // here and now, as above
            }
    };
    struct Step {
        bf16x8_t p[PT], q[2];
    };
    auto prepare = [&](Step& f, const char* X, int s, const u32x4 (&w)[2]) {
#pragma unroll
        for (int t = 0; t < PT; ++t) f.p[t] = fx.read(X, t, s);
#pragma unroll
        for (int n = 0; n < 2; ++n) f.q[n] = weights<ZERO>(w[n][s], zero[n]);
    };
    auto multiply = [&](auto first, const Step& f) {
        const f32x16_t zero = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < PT; ++t)
#pragma unroll
            for (int n = 0; n < 2; ++n)
                acc[t][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f.p[t], f.q[n], decltype(first)::value ? zero : acc[t][n], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
    };
    // this wavefront's LDS reads are back, and all but the last N of its loads have arrived
    auto arrived = [](auto n) {
        constexpr int N = decltype(n)::value;
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        wait_loads<N>();
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
    };
    Step f, h;
    u32x4 w0[2], w1[2];
    uint32_t sc[FOLDS], sn[FOLDS], zc[FOLDS], zn[FOLDS];
    const int pairs = (a.C + 127) / 128;
    if (wave < pairs) {
        load_words(wave);
        __builtin_amdgcn_sched_barrier(0);
        scales(ds, sc, wave);
        if constexpr (ZERO) scales(dz, zc, wave);
        __builtin_amdgcn_sched_barrier(0);
        load_x(xa, wave * 128);
        __builtin_amdgcn_sched_barrier(0);
        load_x(xb, wave * 128 + 64);
        arrived(std::integral_constant<int, 4 * PT>{});
        read_words(w0, 0);
        read_words(w1, 1);
        spread(w0);
        if constexpr (ZERO) group(zc[0]);
        prepare(f, xa, 0, w0);
        // (what lies behind the last pair is fetched as zeros of x)
        for (int p = wave; p < pairs; p += 8) {
            prepare(h, xa, 1, w0);
            multiply(std::true_type{}, f);
            if constexpr (ZERO && FOLDS == 4) group(zc[1]);
            prepare(f, xa, 2, w0);
            multiply(std::false_type{}, h);
            if (FOLDS == 4) fold(sc[0]);
            prepare(h, xa, 3, w0);
            multiply(std::integral_constant<bool, FOLDS == 4>{}, f);
            arrived(std::integral_constant<int, 63>{});         // the reads: words and xa are free
            load_words(p + 8);
            __builtin_amdgcn_sched_barrier(0);
            scales(ds, sn, p + 8);
            if constexpr (ZERO) scales(dz, zn, p + 8);
            __builtin_amdgcn_sched_barrier(0);
            load_x(xa, (p + 8) * 128);
            arrived(std::integral_constant<int, 4 + (ZERO ? 2 : 1) * FOLDS + 4 * PT>{});      // xb
            spread(w1);
            if constexpr (ZERO && FOLDS > 1) group(zc[FOLDS / 2]);
            prepare(f, xb, 0, w1);
            multiply(std::false_type{}, h);
            if (FOLDS > 1) fold(sc[FOLDS == 2 ? 0 : 1]);
            prepare(h, xb, 1, w1);
            multiply(std::integral_constant<bool, (FOLDS > 1)>{}, f);
            if constexpr (ZERO && FOLDS == 4) group(zc[3]);
            prepare(f, xb, 2, w1);
            multiply(std::false_type{}, h);
            if (FOLDS == 4) fold(sc[FOLDS / 2]);
            prepare(h, xb, 3, w1);
            multiply(std::integral_constant<bool, FOLDS == 4>{}, f);
            arrived(std::integral_constant<int, 63>{});
            load_x(xb, (p + 8) * 128 + 64);
            arrived(std::integral_constant<int, 4 * PT>{});     // the next pair's words, scales and xa
            read_words(w0, 0);
            read_words(w1, 1);
            spread(w0);
            if constexpr (ZERO) group(zn[0]);
            prepare(f, xa, 0, w0);
            multiply(std::false_type{}, h);
            fold(sc[FOLDS - 1]);
#pragma unroll
            for (int i = 0; i < FOLDS; ++i) {
                sc[i] = sn[i];
                if constexpr (ZERO) zc[i] = zn[i];
            }
        }
        wait_loads<0>();
    }
    // partial sums [row of x][64 weight rows], 256 bytes a row, half of the rows in either buffer of the
    // wavefront's own.  Register v of a tile: row 8 (v / 4) + 4 (lane / 32) + v % 4 of x, weight row lane & 31.
#pragma unroll
    for (int t = 0; t < PT; ++t)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                const int m = t * 32 + 8 * (v >> 2) + 4 * (lane >> 5) + (v & 3);
                char* half = PT == 2 ? (t ? xb : xa) : (v >> 3 ? xb : xa);
                reinterpret_cast<float*>(half)[m % (kRows / 2) * 64 + n * 32 + (lane & 31)] = total[t][n][v];
            }
    __syncthreads();
    // 8 threads a row of x
    const int m = threadIdx.x >> 3, c = (threadIdx.x & 7) * 8, r = r0 + c;
    if (m >= xrows || r >= a.R) return;
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = 0.0f;
    const char* from = (m < kRows / 2 ? XA : XB) + (m % (kRows / 2) * 64 + c) * 4;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
        const f32x4_t lo = *reinterpret_cast<const f32x4_t*>(from + w * kXBytes);
        const f32x4_t hi = *reinterpret_cast<const f32x4_t*>(from + w * kXBytes + 16);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            v[k] += lo[k];
            v[k + 4] += hi[k];
        }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] *= kNibbleUnit;
    if (vec) store_y8(a, m0 + m, r, v, load_bias8(a, r), load_residual8(a, m0 + m, r));
    else
        for (int k = 0; k < 8 && r + k < a.R; ++k) store_y(a, m0 + m, r + k, v[k]);
}

// Groups that are not multiples of 32 columns (any shape and alignment): 64 x 64 outputs per workgroup,
// four wavefronts of 32 x 32,
// 32 columns a step through LDS; a step never crosses the end of a group (its rest is zero).
template <bool ZERO>
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
                        const int nibble = (int)((word >> (4 * (c % 8))) & 15u);
                        const int z = ZERO ? a.zero[(int64_t)(r0 + row) * a.G + g] : 8;
                        wv = f32_to_bf16_bits((float)(((nibble + z + 8) & 15) - z));     // code - zero
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

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Which kernel (us, C = 7168, R = 4096; 256 workgroups run at a time).  int4_few_kernel, for a few rows of x:
// 1 row 10.5 against 20 of int4_split_kernel<1>, 16 rows 14 / 21.
constexpr int64_t kFewRows = 16;
// int4_split_kernel with 32 rows while its workgroups run at once: 128 rows 21 against 27 with 64 rows, 256
// rows 39 / 29.  And int4_tile_kernel when that one's workgroups would take more than three turns: 512 rows (512
// workgroups) 51 against 95, 768 rows 74 / 100, 1024 rows 101 / 103, 1536 rows 169 / 113; R = 7168, C = 2048, 384 rows
// (672) 32 / 37, 512 rows (896) 41 / 37.
constexpr int64_t kAtOnce = 256, kSplitWorkgroups = 768;
int64_t split_workgroups(int64_t M, int64_t R, int64_t rows) { return forge::ceil_div(R, 64) * forge::ceil_div(M, rows); }

template <int PT, bool ZERO>
void launch_split(const Int4Args& a, bool one_group, bool vec, hipStream_t st) {
    const int r_tiles = (int)forge::ceil_div(a.R, 64), m_tiles = (int)forge::ceil_div(a.M, 32 * PT);
    const dim3 grid((unsigned)(forge::ceil_div((int64_t)r_tiles * m_tiles, 8) * 8));
    if (a.gs % 128 == 0 || one_group) int4_split_kernel<PT, 1, ZERO><<<grid, 512, 0, st>>>(a, r_tiles, m_tiles, vec);
    else if (a.gs % 64 == 0) int4_split_kernel<PT, 2, ZERO><<<grid, 512, 0, st>>>(a, r_tiles, m_tiles, vec);
    else int4_split_kernel<PT, 4, ZERO><<<grid, 512, 0, st>>>(a, r_tiles, m_tiles, vec);
}

template <bool ZERO>
void launch_few(const Int4Args& a, bool one_group, hipStream_t st) {
    const dim3 grid((unsigned)forge::ceil_div(a.R, 16));
    if (a.gs % 128 == 0 || one_group) int4_few_kernel<4, ZERO><<<grid, 512, 0, st>>>(a);
    else if (a.gs % 64 == 0) int4_few_kernel<2, ZERO><<<grid, 512, 0, st>>>(a);
    else int4_few_kernel<1, ZERO><<<grid, 512, 0, st>>>(a);
}

template <bool ZERO>
int launch(const char* name, const Int4Args& a, bool pieces, bool one_group, bool vec, hipStream_t st) {
    const int64_t M = a.M, R = a.R;
    if (!pieces) {
        const int64_t r_tiles = forge::ceil_div(R, 64), blocks = r_tiles * forge::ceil_div(M, 64);
        FORGE_REQUIRE(blocks <= forge::max_workgroups(256), "%s: %lld workgroups, too many for one launch", name, (long long)blocks);
        int4_any_kernel<ZERO><<<dim3((unsigned)blocks), 256, 0, st>>>(a, (int)r_tiles);
    } else if (M <= kFewRows) {
        launch_few<ZERO>(a, one_group, st);
    } else if (split_workgroups(M, R, 32) <= kAtOnce) {
        launch_split<1, ZERO>(a, one_group, vec, st);
    } else if (split_workgroups(M, R, 64) <= kSplitWorkgroups) {
        launch_split<2, ZERO>(a, one_group, vec, st);
    } else {
        const int64_t r_tiles = forge::ceil_div(R, 256), m_tiles = forge::ceil_div(M, 128);
        const int64_t blocks = forge::ceil_div(r_tiles * m_tiles, 8) * 8;
        FORGE_REQUIRE(blocks <= forge::max_workgroups(512), "%s: %lld workgroups, too many for one launch", name, (long long)blocks);
        const dim3 grid((unsigned)blocks);
        if (a.gs % 128 == 0 || one_group) int4_tile_kernel<1, ZERO><<<grid, 512, 0, st>>>(a, (int)r_tiles, (int)m_tiles, vec);
        else if (a.gs % 64 == 0) int4_tile_kernel<2, ZERO><<<grid, 512, 0, st>>>(a, (int)r_tiles, (int)m_tiles, vec);
        else int4_tile_kernel<4, ZERO><<<grid, 512, 0, st>>>(a, (int)r_tiles, (int)m_tiles, vec);
    }
    FORGE_LAUNCH_CHECK();
    return FORGE_OK;
}

int linear_int4(const char* name, const void* x, int64_t ldx, const int32_t* packed, const float* scale,
                const int32_t* zero, bool zeros, int64_t gs, const void* bias, const void* residual, int64_t ldr,
                int64_t M, int64_t C, int64_t R, int act, void* y, forge_stream_t stream) {
    FORGE_REQUIRE(M >= 0 && C >= 1 && R >= 1 && gs >= 1, "%s: M=%lld C=%lld R=%lld gs=%lld", name, (long long)M,
                  (long long)C, (long long)R, (long long)gs);
    FORGE_REQUIRE(M <= (1 << 30) && C <= (1 << 24) && R <= (1 << 24), "%s: M=%lld C=%lld R=%lld: too large "
                  "(M up to 2^30, C and R up to 2^24)", name, (long long)M, (long long)C, (long long)R);
    FORGE_REQUIRE(act >= FORGE_ACT_NONE && act <= FORGE_ACT_RELU, "%s: act=%d", name, act);
    if (M == 0) return FORGE_OK;
    FORGE_REQUIRE(x && packed && scale && y && (zero || !zeros), "%s: null pointer", name);
    FORGE_REQUIRE(ldx >= C && (!residual || ldr >= R), "%s: row pitch %lld / %lld below C=%lld / R=%lld", name,
                  (long long)ldx, (long long)ldr, (long long)C, (long long)R);
    if (gs > C) gs = C;
    Int4Args a{(const uint16_t*)x, (const uint32_t*)packed, scale, zero, (const uint16_t*)bias,
               (const uint16_t*)residual, (uint16_t*)y, ldx, ldr, (int)M, (int)C, (int)R,
               (int)forge::ceil_div(C, gs), (int)gs, (int)forge::ceil_div(C, 8), act};
    hipStream_t st = (hipStream_t)stream;
    forge::KernelTiming timing(name + 6, st, 2.0 * M * C * R, forge::WORK_FLOPS);
    const bool one_group = a.G == 1;
    const bool pieces = C % 8 == 0 && ldx % 8 == 0 && ldx < (1 << 21) && aligned16(x) &&
                        (gs % 32 == 0 || one_group);
    const bool vec = R % 8 == 0 && aligned16(y) && aligned16(bias) && aligned16(residual) && (!residual || ldr % 8 == 0);
    return zeros ? launch<true>(name, a, pieces, one_group, vec, st) : launch<false>(name, a, pieces, one_group, vec, st);
}
}  // namespace

extern "C" int forge_linear_int4(const void* x, int64_t ldx, const int32_t* packed, const float* scale,
                                 int64_t gs, const void* bias, const void* residual, int64_t ldr, int64_t M,
                                 int64_t C, int64_t R, int act, void* y, forge_stream_t stream) {
    return linear_int4("forge_linear_int4", x, ldx, packed, scale, nullptr, false, gs, bias, residual, ldr, M, C, R,
                       act, y, stream);
}

extern "C" int forge_linear_int4_zeros(const void* x, int64_t ldx, const int32_t* packed, const float* scale,
                                       const int32_t* zero, int64_t gs, const void* bias, const void* residual,
                                       int64_t ldr, int64_t M, int64_t C, int64_t R, int act, void* y,
                                       forge_stream_t stream) {
    return linear_int4("forge_linear_int4_zeros", x, ldx, packed, scale, zero, true, gs, bias, residual, ldr, M, C,
                       R, act, y, stream);
}
