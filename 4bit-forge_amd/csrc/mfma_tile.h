// 256 x 256 tiles of a bf16 product for the 32x32x16 matrix instruction: how a 64-deep stage of
// either operand lies in LDS, how it gets there, and how a wavefront reads its fragments.
//
// A workgroup is 8 wavefronts, 2 along P (the operand that runs along the accumulator's registers)
// by 4 along Q (the one that runs across the lanes): 128 x 64 outputs each, 8 matrix instructions
// per 6 fragments.  Per stage that is 192 KB of LDS reads for 2048 clocks of matrix work at 128
// bytes a clock, so the matrix pipe and not the LDS is the limit; 64 x 64 per wavefront (16
// wavefronts) would need 256 KB and sit exactly on it.
//
// A stage is 64 deep; the 160 KB of LDS are three buffers of P and two of Q.  Stages go from memory to LDS
// without touching registers (buffer_load ... lds, 16 bytes a lane), issued as soon as their buffer has been
// read: Q's a stage before their use, P's two (with two buffers of P, 128 KB, a stage that comes from HBM
// arrives too late: 16 experts at 7168 x 2048 and 16384 rows took 950 us and now 855, one expert at 7168 x 1024
// and 32768 rows 768 and now 722, 1334 TFLOP/s).  A lane whose element lies outside the matrix gets an
// offset beyond the descriptor's range, for which the hardware writes zeros; stages behind the last
// are fetched like that too.
//
// The lanes of one such load write 1 KiB of consecutive LDS, so the layout that keeps the reads free of
// bank conflicts is made by choosing which 16 bytes each lane fetches:
//   K_INNER (the inner dimension is contiguous in memory): 256 rows of 128 bytes; 16-byte piece c of
//     row r lies at piece c ^ (r / 2 % 8), so 16 consecutive rows of one piece cover all 64 banks.
//     (Stages of 32 with four buffers were slower: rows of 64 bytes are twice the L2 requests.)
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
// all but the last N of this wavefront's loads have arrived, and all of its LDS reads (vmcnt(N), lgkmcnt(0))
template <int N>
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | ((N >> 4) << 14)); }
// the same, then the workgroup's barrier; nothing the compiler knows of moves across it
template <int N>
__device__ __forceinline__ void wait_loads_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    wait_loads<N>();
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
}

// ---- K_INNER: the descriptor covers exactly the valid rows of pitch ld, so that rows behind them are
// outside its range; the columns from `inner` on are sorted out here.  A wavefront has LOADS loads of 8
// rows (an even number), load j 8 j rows behind its first; its lanes' pieces are those of load 0 for even j, and the
// others of their 128 bytes (piece ^ 4) for odd j.
template <int LOADS>
struct InnerLoader {
    uint32_t off;        // byte offset of this lane's row, load 0
    int piece;           // columns into the stage, load 0
    // first_row: which row of the descriptor the wavefront's first row is
    __device__ __forceinline__ void init(int lane, int64_t ld, int first_row) {
        off = (uint32_t)((first_row + lane / 8) * ld * 2);
        piece = ((lane & 7) ^ (lane >> 4)) * 8;
    }
    __device__ __forceinline__ void stage(__amdgpu_buffer_rsrc_t d, char* lds, int wave, int64_t ld, int k0, int inner) const {
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const int k = k0 + ((j & 1) ? piece ^ 32 : piece);
            load_to_lds(d, lds + (wave * LOADS + j) * 1024, k < inner ? off + (uint32_t)(k * 2) + (uint32_t)(j * 16 * ld) : kOutside);
        }
    }
};
// ---- K_OUTER: columns `col0 ..` of a matrix whose rows are the inner dimension.  The descriptor is
// made per stage (base at the stage's first row), so row offsets never pass 32 bits.
template <int DEPTH = kStage>
struct OuterLoader {
    static constexpr int kLoads = DEPTH / 16;      // of a wavefront, two rows each
    uint32_t even, odd;  // byte offsets of loads 0 and 1; 2 and 3 are 4 rows behind
    __device__ __forceinline__ void init(int wave, int lane, int64_t ld, int cols) {
        const int k = wave * 2 * kLoads + lane / 32, c = (lane & 31) ^ ((lane / 32) << 2);
        even = c * 8 < cols ? (uint32_t)(k * ld * 2) + c * 16 : kOutside;
        odd = (c ^ 8) * 8 < cols ? (uint32_t)((k + 2) * ld * 2) + (c ^ 8) * 16 : kOutside;
    }
    // base: first row of the stage at the tile's first column; rows left in the matrix from there
    __device__ __forceinline__ void stage(const uint16_t* base, int64_t ld, int left, int cols, char* lds, int wave) const {
        const int rows = min(left, DEPTH), width = min(cols, kTile);
        const int size = max((rows - 1) * (int)ld + width, 0);           // 0 rows or fewer: nothing
        const __amdgpu_buffer_rsrc_t d = descriptor(base, (uint32_t)size * 2);
#pragma unroll
        for (int j = 0; j < kLoads; ++j)
            // (kOutside plus a few rows is still outside)
            load_to_lds(d, lds + (wave * kLoads + j) * 1024, ((j & 1) ? odd : even) + (uint32_t)((j >> 1) * 8 * ld));
    }
};

// ---- fragments: 32 rows (tile t of the operand) x 16 of the inner dimension (step s of the stage)
struct InnerFragment {
    static constexpr int kReads = 1;     // LDS instructions per fragment
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
    static constexpr int kReads = 2;
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

// The fragments of one step: NP of P (every SKIP-th), NQ of Q
template <int NP, int NQ = 2, int SKIP = 1>
struct Fragments {
    bf16x8_t p[NP], q[NQ];
    template <typename FP, typename FQ>
    __device__ __forceinline__ void read(const char* P, const char* Q, const FP& fp, const FQ& fq, int s) {
#pragma unroll
        for (int t = 0; t < NQ; ++t) q[t] = fq.read(Q, t, s);
#pragma unroll
        for (int t = 0; t < NP; ++t) p[t] = fp.read(P, t * SKIP, s);
    }
    __device__ __forceinline__ void multiply(f32x16_t (&acc)[NP][NQ]) const {
#pragma unroll
        for (int t = 0; t < NP; ++t)
#pragma unroll
            for (int n = 0; n < NQ; ++n)
                acc[t][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(p[t], q[n], acc[t][n], 0, 0, 0);
    }
};

// The order in which a step issues: after every matrix instruction its share of the next step's LDS
// reads and (LOADS) of the loads to LDS.  Left alone the compiler sinks the reads to the step's end.
template <int READS, int LOADS>
__device__ __forceinline__ void order_step() {
    constexpr int kPer = (READS + 5) / 6;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                       // matrix instruction
        if (i < LOADS) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);        // load to LDS
        if (i < 6) __builtin_amdgcn_sched_group_barrier(0x100, kPer, 0);         // LDS read
    }
}

// The inner loop.  load_p(s, P) and load_q(s, Q) issue stage s's loads (4 each per wavefront).  A stage is
// four steps; while a step's 8 matrix instructions run, the next step's fragments are read.  The one
// barrier of a stage sits before its last step, whose fragments are in registers by then: nothing waits
// behind it.  It publishes that the next stage has arrived and that this stage's buffers have been read, which
// the loads of Q's stage after next, and a step later of P's third next, then fill.  Loads return in the
// order of their issue, so the wait is for all but the youngest four.
// The buffers are separate arrays and the loop is unrolled over them because the compiler otherwise
// has to assume that a load on its way to LDS may hit what is being read, and waits for it.
template <typename LOADP, typename LOADQ, typename FP, typename FQ>
__device__ __forceinline__ void one_stage(int s, const char* P, char* Q, const char* Pn, const char* Qn, char* Pl, LOADP& load_p, LOADQ& load_q,
                                          const FP& fp, const FQ& fq, Fragments<4>& f, f32x16_t (&acc)[4][2]) {
    constexpr int kReads = 4 * FP::kReads + 2 * FQ::kReads;
    Fragments<4> g;
    load_p(s + 2, Pl);
    g.read(P, Q, fp, fq, 1);
    f.multiply(acc);
    order_step<kReads, 4>();
    __builtin_amdgcn_sched_barrier(0);
    f.read(P, Q, fp, fq, 2);
    g.multiply(acc);
    order_step<kReads, 0>();
    __builtin_amdgcn_sched_barrier(0);
    g.read(P, Q, fp, fq, 3);
    f.multiply(acc);
    order_step<kReads, 0>();
    wait_loads_barrier<4>();
    load_q(s + 2, Q);
    f.read(Pn, Qn, fp, fq, 0);
    g.multiply(acc);
    order_step<kReads, 4>();
    __builtin_amdgcn_sched_barrier(0);
}

// stages >= 1
template <typename LOADP, typename LOADQ, typename FP, typename FQ>
__device__ __forceinline__ void multiply_stages(int stages, char* P0, char* P1, char* P2, char* Q0, char* Q1, LOADP& load_p, LOADQ& load_q,
                                                const FP& fp, const FQ& fq, f32x16_t (&acc)[4][2]) {
    load_p(0, P0);
    load_q(0, Q0);
    __builtin_amdgcn_sched_barrier(0);
    load_p(1, P1);
    load_q(1, Q1);
    wait_loads_barrier<8>();
    Fragments<4> f;
    f.read(P0, Q0, fp, fq, 0);
    int s = 0;
    for (; s + 6 <= stages; s += 6) {
        one_stage(s, P0, Q0, P1, Q1, P2, load_p, load_q, fp, fq, f, acc);
        one_stage(s + 1, P1, Q1, P2, Q0, P0, load_p, load_q, fp, fq, f, acc);
        one_stage(s + 2, P2, Q0, P0, Q1, P1, load_p, load_q, fp, fq, f, acc);
        one_stage(s + 3, P0, Q1, P1, Q0, P2, load_p, load_q, fp, fq, f, acc);
        one_stage(s + 4, P1, Q0, P2, Q1, P0, load_p, load_q, fp, fq, f, acc);
        one_stage(s + 5, P2, Q1, P0, Q0, P1, load_p, load_q, fp, fq, f, acc);
    }
    if (s < stages) one_stage(s, P0, Q0, P1, Q1, P2, load_p, load_q, fp, fq, f, acc);
    if (s + 1 < stages) one_stage(s + 1, P1, Q1, P2, Q0, P0, load_p, load_q, fp, fq, f, acc);
    if (s + 2 < stages) one_stage(s + 2, P2, Q0, P0, Q1, P1, load_p, load_q, fp, fq, f, acc);
    if (s + 3 < stages) one_stage(s + 3, P0, Q1, P1, Q0, P2, load_p, load_q, fp, fq, f, acc);
    if (s + 4 < stages) one_stage(s + 4, P1, Q0, P2, Q1, P0, load_p, load_q, fp, fq, f, acc);
    // loads of stages behind the last (zeros) are still on their way to LDS: a workgroup that ends
    // gives its LDS away
    wait_loads<0>();
}

// The same where both operands are K_OUTER, for tiles that follow one another without a pause (the loads go on across
// the border): stages of 32 with four buffers of either, fetched three stages ahead.  Half as deep would be half as
// many bytes of a row where the inner dimension is contiguous; here a row's 512 bytes stay together.
// load() issues the loads that this stage's buffers are to get (4 per wavefront); YOUNGER is how many loads and
// stores were issued behind those of the next stage, which are all that is waited for.
constexpr int kShort = 32;
template <int YOUNGER, typename LOAD, typename FP, typename FQ>
__device__ __forceinline__ void one_short_stage(const char* P, const char* Q, const char* Pn, const char* Qn, LOAD load, const FP& fp,
                                                const FQ& fq, Fragments<4>& f, f32x16_t (&acc)[4][2]) {
    constexpr int kReads = 4 * FP::kReads + 2 * FQ::kReads;
    Fragments<4> g;
    g.read(P, Q, fp, fq, 1);
    f.multiply(acc);
    order_step<kReads, 0>();
    wait_loads_barrier<YOUNGER>();
    load();
    f.read(Pn, Qn, fp, fq, 0);
    g.multiply(acc);
    order_step<kReads, 4>();
    __builtin_amdgcn_sched_barrier(0);
}

// What a wavefront without outputs of its own does meanwhile: its share of the loads, and the barriers
template <typename LOADP, typename LOADQ>
__device__ __forceinline__ void load_stages(int stages, char* P0, char* P1, char* P2, char* Q0, char* Q1, LOADP& load_p, LOADQ& load_q) {
    load_p(0, P0);
    load_q(0, Q0);
    __builtin_amdgcn_sched_barrier(0);
    load_p(1, P1);
    load_q(1, Q1);
    wait_loads_barrier<8>();
    auto stage = [&](int s, char* Q, char* Pl) {
        load_p(s + 2, Pl);
        wait_loads_barrier<4>();
        load_q(s + 2, Q);
        __builtin_amdgcn_sched_barrier(0);
    };
    int s = 0;
    for (; s + 6 <= stages; s += 6) {
        stage(s, Q0, P2);
        stage(s + 1, Q1, P0);
        stage(s + 2, Q0, P1);
        stage(s + 3, Q1, P2);
        stage(s + 4, Q0, P0);
        stage(s + 5, Q1, P1);
    }
    if (s < stages) stage(s, Q0, P2);
    if (s + 1 < stages) stage(s + 1, Q1, P0);
    if (s + 2 < stages) stage(s + 2, Q0, P1);
    if (s + 3 < stages) stage(s + 3, Q1, P2);
    if (s + 4 < stages) stage(s + 4, Q0, P0);
    wait_loads<0>();
}

// Tiles with up to 64 rows of Q: bound by P's bytes, so its loads go out a stage earlier, three ahead.
// Q's stages are 8 KB; wavefront w has 32 rows of Q (w / 4) and two tiles of P; load_q issues one load.
template <int SKIP, typename LOADP, typename LOADQ, typename FP, typename FQ>
__device__ __forceinline__ void one_light_stage(int s, char* P, char* Q, LOADP& load_p, LOADQ& load_q, const FP& fp, const FQ& fq, f32x16_t (&acc)[2][1]) {
    Fragments<2, 1, SKIP> f[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) f[k].read(P, Q, fp, fq, k);
    wait_loads_barrier<4>();                 // this stage has been read; the next one is here (its third next's P is not)
    load_q(s + 2, Q);
    __builtin_amdgcn_sched_barrier(0);
    load_p(s + 3, P);
#pragma unroll
    for (int k = 0; k < 4; ++k) f[k].multiply(acc);
}
template <int SKIP, typename LOADP, typename LOADQ, typename FP, typename FQ>
__device__ __forceinline__ void multiply_light_stages(int stages, char* P0, char* P1, char* P2, char* Q0, char* Q1, LOADP& load_p, LOADQ& load_q,
                                                      const FP& fp, const FQ& fq, f32x16_t (&acc)[2][1]) {
    load_p(0, P0);
    load_q(0, Q0);
    __builtin_amdgcn_sched_barrier(0);
    load_p(1, P1);
    load_q(1, Q1);
    __builtin_amdgcn_sched_barrier(0);
    load_p(2, P2);
    wait_loads_barrier<9>();
    int s = 0;
    for (; s + 6 <= stages; s += 6) {
        one_light_stage<SKIP>(s, P0, Q0, load_p, load_q, fp, fq, acc);
        one_light_stage<SKIP>(s + 1, P1, Q1, load_p, load_q, fp, fq, acc);
        one_light_stage<SKIP>(s + 2, P2, Q0, load_p, load_q, fp, fq, acc);
        one_light_stage<SKIP>(s + 3, P0, Q1, load_p, load_q, fp, fq, acc);
        one_light_stage<SKIP>(s + 4, P1, Q0, load_p, load_q, fp, fq, acc);
        one_light_stage<SKIP>(s + 5, P2, Q1, load_p, load_q, fp, fq, acc);
    }
    if (s < stages) one_light_stage<SKIP>(s, P0, Q0, load_p, load_q, fp, fq, acc);
    if (s + 1 < stages) one_light_stage<SKIP>(s + 1, P1, Q1, load_p, load_q, fp, fq, acc);
    if (s + 2 < stages) one_light_stage<SKIP>(s + 2, P2, Q0, load_p, load_q, fp, fq, acc);
    if (s + 3 < stages) one_light_stage<SKIP>(s + 3, P0, Q1, load_p, load_q, fp, fq, acc);
    if (s + 4 < stages) one_light_stage<SKIP>(s + 4, P1, Q0, load_p, load_q, fp, fq, acc);
    wait_loads<0>();
}

// Workgroup b of a launch runs on XCD b % 8 (each has its own L2).  Of `tiles` tiles every XCD takes
// a run of consecutive ones, so that tiles that share an operand share an L2; the tile of b's, or
// `tiles` or more if there is none.
__device__ __forceinline__ int xcd_tile(int b, int tiles) {
    const int per = (tiles + 7) / 8, i = b / 8;
    return i < per ? (b % 8) * per + i : tiles;
}

// The same for two lists, `full` tiles that take long and `light` ones that take little matrix work but as many
// bytes: every XCD takes an eighth of either list.  The light ones lie evenly between the others, so
// that the memory is in use all the time, but for the last 32, which even out the end.  True and t: a full tile;
// false: a light one (t = light or more: none).  Launch 8 workgroups more than there are tiles, rounded up to 8.
__device__ __forceinline__ bool xcd_tile(int b, int full, int light, int& t) {
    const int x = b % 8, i = b / 8;
    const int f0 = min(x * ((full + 7) / 8), full), fn = min((x + 1) * ((full + 7) / 8), full) - f0;
    const int l0 = min(x * ((light + 7) / 8), light), ln = min((x + 1) * ((light + 7) / 8), light) - l0;
    const int n = fn + max(ln - 32, 0);
    if (i >= n) {
        t = i - fn < ln ? l0 + i - fn : light;
        return false;
    }
    const int before = (int)(((int64_t)i * fn + n - 1) / n), upto = (int)(((int64_t)(i + 1) * fn + n - 1) / n);
    t = upto > before ? f0 + before : l0 + i - before;
    return upto > before;
}

}  // namespace forge
