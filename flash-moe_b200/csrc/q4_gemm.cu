// Products of 4-bit affine matrices with many tokens: projections of a prompt, and the routed experts once an expert sees
// more than a handful of tokens.  tcgen05 / TMEM / TMA.
//
// Reference: dequant_gemm_4bit_batch (metal_infer/shaders.metal) and, per expert, the chain of metal_infer/gpu_dispatch.h.
//     y[r][t] = sum_g sum_{k in g} s[r][g] (nibble[r][k] - 8) x[t][k]  +  sum_g (b[r][g] + 8 s[r][g]) X[t][g]
// with X[t][g] the sum of the group's 64 inputs.
//
// Exactness.  A scale is bf16 (8 bits) and |nibble - 8| is 8 or has 3 bits, so s * (nibble - 8) has 11 bits at most: it
// IS an fp16 number, once a power of two per row and 256 inputs has brought the scales into range.  Scales down to 1/128 of the
// largest of their 256 inputs take one multiply-add; where a warp has smaller ones, a second multiplication takes them in down to
// 2^-23, and what lies below keeps an absolute error of 2^-31 of the largest per weight.  An activation enters
// as two fp16 terms, hi + lo, under a power of two per token: 22 bits down to 2^-16 of the token's largest, below that an absolute
// error of 2^-39 of it (a sum X: 2^-33).  The second sum is one more block of 64 columns, per 64 groups, with both factors in two
// terms: b + 8 s keeps 22 bits down to 2^-16 of the largest of its row's 64, below that an absolute error of 2^-39 of it.  (b and
// 8 s by themselves would be exact further down, but that block needs both at once, and the registers it spilled cost the experts
// 2 %.)  The tensor cores add into fp32 by truncation, which shrinks a long sum by a
// few 2^-24 per addition; so TMEM accumulates over 256 inputs only, and the parts are added in fp32 by the epilogue
// warps, which apply the row's power of two in the same fused multiply-add.
//
// Organisation (persistent, one CTA per SM).  A unit is two row tiles of 128 rows (kGateUp: the same rows of gate and up, so
// that SwiGLU needs no exchange) and up to 96 tokens; a step is one tile over one chunk of 4 groups.
//   warps 0-7    widen: a thread owns a row; two 16-byte reads from the TMA-filled weight tile per group, 9 instructions per word
//                of eight nibbles, 32 TMEM columns per store.  Operand A lives in TMEM: written row by row where the MMA wants
//                it, and an MMA of N = 96 takes 57 cycles from there, 87 from shared memory.
//   warps 8-15   epilogue: running sums in TMEM, added up per step; the last step of a tile writes the results, 128
//                consecutive features per token and store
//   warps 16, 18 TMA producers of token tiles (two groups, hi | lo each) and of weight tiles [128 rows][128 bytes]
//   warps 17, 19 issue the MMAs of a tile each (M128, N = the unit's tokens rounded up to 16, K16): while one waits, the other's
//                keep the tensor core busy
// TMEM columns: 2 * 96 of steps in flight, 2 * 96 running sums, 2 * 64 operand A (two slots of two groups).
// Why 96: sums, steps and operands share 512 columns, token tiles 144 KB; at 64 tokens a weight is widened half as often again
// and the MMA's start-up counts more, at 128 the steps could not be double-buffered.
//
// Measured (B200; the tensor work is twice the product's, because of the two terms): 4096 tokens x 4096 x 8192 in 520 us as a
// replayed graph, 528 TFLOP/s of products (the tensor core is busy 72 % of the time in MMAs of 57 cycles, ideal 48), 610 us in calls
// on fresh inputs (450 TFLOP/s, under the power cap); 300 tokens through qkv + z + beta + alpha of 4096 in 117 and 132 us; 4096
// tokens through 10 of 512 experts of 4096 x 1024: gate / up 1.77 ms, down 0.98 ms.
// What bounds it: the issue slots.  Widening, the epilogue and the hand-overs between the roles take 2000 to 2300 instructions
// per operand slot of 915 tensor cycles; below 64 tokens a unit takes about 950 cycles per slot whatever its tokens.
// Tried and not kept: 16 widening warps (the same time), the two issuing warps as one (+10 %), operand slots of one group
// (+12 %), gathering token rows with tile::gather4 instead of in the split (+30 % of the gate / up launch).
// Every wait is bounded; on expiry the CTA records an error code and winds down.
#include <cuda.h>
#include <cuda_fp16.h>

#include <string.h>

#include <algorithm>

#include "fm_device.cuh"
#include "fm_internal.h"
#include "fm_tc.cuh"

namespace fm {

namespace {

constexpr int kTok = kGemmTokens;           // tokens per unit (96)
constexpr int kChunk = 4;                   // groups per step
constexpr int kBTile = kTok * 128;          // bytes of a token tile: one group, one term
constexpr int kBSlot = 4 * kBTile;          // two groups, hi then lo each
constexpr int kBSlots = 3;
constexpr int kWSlot = 128 * 128;           // bytes of a weight tile: 128 rows, 4 groups
constexpr int kWSlots = 4;
constexpr int kGemmThreads = 20 * 32;
constexpr int T = 2;                        // row tiles of a unit
constexpr float kSumScale = 0x1p-6f;        // of the stored sums of 64 inputs
constexpr int kDBufs = T;                   // steps in flight: one per tile
// Steps whose row factors are kept: the widening warps are at most the operand slots (one to a step at the least), the
// steps in flight and their own step ahead of the epilogue.
constexpr int kFSteps = 16;
constexpr int kHalf = kTok / 2;            // columns of an epilogue warp
constexpr uint32_t kColStep = 0, kColSum = kDBufs * kTok;  // TMEM columns; operand A behind the sums

constexpr uint32_t kColA = kColSum + T * kTok;
static_assert(kColA + 128 <= 512, "two operand slots of two groups each");
constexpr int kA = 2;                       // operand slots

enum Bar { BAR_W_FULL = 0, BAR_W_EMPTY = BAR_W_FULL + kWSlots, BAR_B_FULL = BAR_W_EMPTY + kWSlots, BAR_B_EMPTY = BAR_B_FULL + kBSlots,
           BAR_D_FULL = BAR_B_EMPTY + kBSlots, BAR_D_EMPTY = BAR_D_FULL + kDBufs, BAR_A_FULL = BAR_D_EMPTY + kDBufs,
           BAR_A_EMPTY = BAR_A_FULL + 8, BAR_END = BAR_A_EMPTY + 8, BAR_COUNT = BAR_END + 2 };
constexpr int kGemmSmem = kBSlots * kBSlot + kWSlots * kWSlot + kFSteps * 128 * 4 + BAR_COUNT * 8 + 1024;

struct GemmMaps {
    CUtensorMap w[kMaxProj];  // words: [matrix][rows][K / 8] (kGateUp: 0 gate, 1 up)
    CUtensorMap s[kMaxProj], b[kMaxProj];  // scales and biases [matrix][rows][K / 64], where wide (groups a multiple of 8, 16-byte aligned)
    CUtensorMap x;            // fp16 [rows][hi | lo]
};
struct GemmParams {
    Q4Params p;
    int G, pseudo, units_per_job, kp;  // groups, blocks of 64 groups, row units, columns of one term of x
    int m_units[kMaxProj];             // kProj: row units of each matrix
    const float *tscale;               // what a row of x has to be multiplied with
    int *err;
};

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
                 : "memory");
}
// 32 lanes x 16 consecutive 32-bit columns
__device__ __forceinline__ void tc_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr)
                 : "memory");
}
// True in one lane of the warp, the same one for every call.
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(one));
    return one != 0;
}

// The same value in every lane, and known to the compiler as such (values of at least 0).
__device__ __forceinline__ int uniform(int v) { return __reduce_max_sync(0xffffffffu, v); }

// A ring position: slot and the parity its next phase completes with.
template <int N>
struct Ring {
    int slot = 0;
    uint32_t phase = 0;
    __device__ void next() {
        if (++slot == N) { slot = 0; phase ^= 1; }
    }
};

// One unit, as every role works it out for itself.
struct Unit {
    int mat, row0, rows;   // matrix, first row, rows of the matrix
    int expert;
    int tiles;             // row tiles that hold rows; none: the second half of a cut unit of one tile, its CTA's last
    int start, cnt, ncols; // tokens (kProj) or positions in pair_of; columns of the MMA
};

template <Q4Mode MODE, bool WARP = true>
__device__ __forceinline__ Unit unit_at(const GemmParams &g, int u, int whole) {
    Unit r;
    int half = -1;
    if (MODE == kProj && u >= whole) {
        half = (u - whole) & 1;
        u = whole + ((u - whole) >> 1);
    }
    const int job = u / g.units_per_job;
    int mu = u - job * g.units_per_job;
    r.mat = 0; r.expert = 0;
    if constexpr (MODE == kProj) {
        while (mu >= g.m_units[r.mat]) mu -= g.m_units[r.mat++];
        r.start = job * kTok;
        r.cnt = min(kTok, g.p.n - r.start);
    } else {
        const int4 j = g.p.plan.jobs[job];
        if constexpr (WARP) { r.expert = uniform(j.x); r.start = uniform(j.y); r.cnt = uniform(j.z); }
        else { r.expert = j.x; r.start = j.y; r.cnt = j.z; }
    }
    constexpr int kRows = MODE == kGateUp ? T * 64 : T * 128;
    r.row0 = mu * kRows + (half > 0 ? 128 : 0);
    r.rows = g.p.mat[r.mat].rows;
    const int t = (min(half >= 0 ? 128 : kRows, r.rows - r.row0) + 127) / 128;
    r.tiles = MODE == kGateUp ? 2 * t : t;
    r.ncols = (r.cnt + 15) / 16 * 16;
    return r;
}
template <Q4Mode MODE>
__device__ __forceinline__ int tile_row(const Unit &u, int tile) {
    return u.row0 + 128 * (MODE == kGateUp ? tile >> 1 : tile);
}
template <Q4Mode MODE>
__device__ __forceinline__ int tile_mat(const Unit &u, int tile) {
    return MODE == kGateUp ? tile & 1 : u.mat;
}

// The four scales of a row's chunk as bf16 bits, where scales are wide.  Volatile: the load stays where it is written, a step
// ahead of its use.
__device__ __forceinline__ uint2 chunk_scales(const unsigned char *row, int c) {
    uint2 v;
    asm volatile("ld.global.nc.v2.u32 {%0,%1}, [%2];\n" : "=r"(v.x), "=r"(v.y) : "l"(reinterpret_cast<const uint2 *>(row) + c));
    return v;
}
// Where they are not, a row begins at any even address.  It is read in aligned windows, each once, and its pieces are cut out
// of two of them.  Read 2 bytes at a time (a sector of 32 per load and row, next to no L1 beside the tiles) 4160 inputs took
// 2.4 times as long as 4096 (4096 rows, 20 tokens), in windows 1.35 times (28 and 21 us as a replayed graph).  A window that reaches beyond the matrix is
// read by the 2 bytes that belong to it.
struct Bytes { const unsigned char *begin, *end; };
__device__ __forceinline__ uint2 window8(const unsigned char *at, Bytes m) {
    uint2 v = make_uint2(0, 0);
    if (at >= m.begin && at + 8 <= m.end) return chunk_scales(at, 0);
    const uint16_t *h = reinterpret_cast<const uint16_t *>(at);
    const uint16_t *lo = reinterpret_cast<const uint16_t *>(m.begin), *hi = reinterpret_cast<const uint16_t *>(m.end);
    if (h >= lo && h < hi) v.x = __ldg(h);
    if (h + 1 >= lo && h + 1 < hi) v.x |= (uint32_t)__ldg(h + 1) << 16;
    if (h + 2 >= lo && h + 2 < hi) v.y = __ldg(h + 2);
    if (h + 3 >= lo && h + 3 < hi) v.y |= (uint32_t)__ldg(h + 3) << 16;
    return v;
}
// Eight bytes from `by` (0, 2, 4 or 6) bytes into two windows, of which the first `left` halves are kept.
__device__ __forceinline__ uint2 cut8(uint2 a, uint2 b, uint32_t by, int left) {
    const uint32_t w0 = by & 4 ? a.y : a.x, w1 = by & 4 ? b.x : a.y, w2 = by & 4 ? b.y : b.x, s = (by & 2) * 8;
    uint2 v = make_uint2(__funnelshift_r(w0, w1, s), __funnelshift_r(w1, w2, s));
    if (left < 4) v.y &= left < 3 ? 0u : 0xffffu;
    if (left < 2) v.x &= 0xffffu;
    return v;
}
__device__ __forceinline__ uint4 window16(const unsigned char *at) {
    uint4 v;
    asm volatile("ld.global.nc.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(at));
    return v;
}
// The same of 16-byte windows.
__device__ __forceinline__ uint4 cut16(uint4 a, uint4 b, uint32_t by) {
    const bool p = by & 8, q = by & 4;
    const uint32_t t0 = p ? a.z : a.x, t1 = p ? a.w : a.y, t2 = p ? b.x : a.z, t3 = p ? b.y : a.w, t4 = p ? b.z : b.x, t5 = p ? b.w : b.y;
    const uint32_t w0 = q ? t1 : t0, w1 = q ? t2 : t1, w2 = q ? t3 : t2, w3 = q ? t4 : t3, w4 = q ? t5 : t4, s = (by & 2) * 8;
    return make_uint4(__funnelshift_r(w0, w1, s), __funnelshift_r(w1, w2, s), __funnelshift_r(w2, w3, s), __funnelshift_r(w3, w4, s));
}
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("max.u16x2 %0, %1, %2;\n" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint32_t min_u16x2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("min.u16x2 %0, %1, %2;\n" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
// Exponent field of a chunk's largest scale, kept where the powers of two made of it are normal numbers; *far: whether one of
// the four lies below 1/128 of it.  Looking for those costs ordinary matrices 1 % (4096 tokens x 4096 x 8192) to 2 % (4096 tokens
// through 10 of 512 experts); a branch around the whole of the widening cost the experts 3 %.
__device__ __forceinline__ int chunk_exponent(uint2 v, bool *far) {
    const uint32_t a = v.x & 0x7fff7fffu, b = v.y & 0x7fff7fffu;
    uint32_t hi = max_u16x2(a, b), lo = min_u16x2(a, b);
    hi = max(max_u16x2(hi, __byte_perm(hi, 0, 0x1032)), 0x08000800u);  // the same in both halves from here on
    lo = min_u16x2(lo, __byte_perm(lo, 0, 0x1032));
    *far = (int)(hi - lo) > 0x03800380;
    return min((int)(hi >> 23), 244);
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ float pow2(int biased) { return __uint_as_float((uint32_t)biased << 23); }
__device__ __forceinline__ uint32_t h2_bits(__half2 v) { return *reinterpret_cast<const uint32_t *>(&v); }

// (n_q - 8, n_{q+4} - 8) * m * 2^-24 for q = 0..3 of a weight word.  A nibble in the low bits of a half is the subnormal
// fp16 number n * 2^-24 (16 n * 2^-24 one nibble up), so one fused multiply-add takes the 8 off and the scale on, exactly: m
// is the scale as an integer below 2^15 with 8 bits.  A scale below 1/128 of its chunk's largest has less than 8 bits left as
// such an integer.  Where a warp has one, m is 2^15 for all of them, which leaves (n - 8) * 2^-9, and a second multiplication
// takes the scale on.
__device__ __forceinline__ uint32_t fma_h2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;\n" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}
__device__ __forceinline__ void widen_word(uint32_t w, uint32_t m, uint32_t m16, uint32_t c, uint32_t *out) {
    const uint32_t v = w >> 8;
    out[0] = fma_h2(w & 0x000F000Fu, m, c);
    out[1] = fma_h2(w & 0x00F000F0u, m16, c);
    out[2] = fma_h2(v & 0x000F000Fu, m, c);
    out[3] = fma_h2(v & 0x00F000F0u, m16, c);
}
__device__ __forceinline__ uint32_t mul_h2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.f16x2 %0, %1, %2;\n" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
// x as fp16 in both halves
__device__ __forceinline__ uint32_t dup_h2(float x) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %1;\n" : "=r"(d) : "f"(x));
    return d;
}
// (a0, a1) = (a0, a1) * f + (b0, b1) in one instruction
__device__ __forceinline__ void fma_f32x2(uint32_t &a0, uint32_t &a1, uint64_t ff, uint32_t b0, uint32_t b1) {
    uint64_t a, b, d;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(a) : "r"(a0), "r"(a1));
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(b) : "r"(b0), "r"(b1));
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(d) : "l"(a), "l"(ff), "l"(b));
    asm("mov.b64 {%0, %1}, %2;\n" : "=r"(a0), "=r"(a1) : "l"(d));
}

// Bounded wait like mbar_wait, with the thread suspended meanwhile: polling warps take issue slots from the widening ones.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int *abort_flag) {
    long long t0 = 0;
    while (true) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
            : "=r"(done)
            : "r"(bar), "r"(parity), "r"(1000000u)
            : "memory");
        if (done) return true;
        if (*abort_flag) return false;
        if (t0 == 0) t0 = clock64();
        else if (clock64() - t0 > 1000000000LL) {
            *abort_flag = 1;
            return false;
        }
    }
}
template <Q4Mode MODE, bool WIDE>
__global__ void __launch_bounds__(kGemmThreads, 1)
q4_gemm_kernel(const __grid_constant__ GemmMaps maps, const __grid_constant__ GemmParams g) {
    extern __shared__ unsigned char smem_raw[];
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort, s_whole, s_units;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t sB = base, sW = sB + kBSlots * kBSlot;
    float *s_f = reinterpret_cast<float *>(smem_raw + (sW + kWSlots * kWSlot - smem_u32(smem_raw)));  // [steps][128 rows] power of two of the step
    const uint32_t sBar = sW + kWSlots * kWSlot + kFSteps * 128 * 4;
    auto bar = [&](int i) { return sBar + 8u * (uint32_t)i; };
    const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;
    if (tid == 0) {
        s_abort = 0;
        for (int i = 0; i < kWSlots; i++) { mbar_init(bar(BAR_W_FULL + i), 1); mbar_init(bar(BAR_W_EMPTY + i), 8); }
        for (int i = 0; i < kBSlots; i++) { mbar_init(bar(BAR_B_FULL + i), 1); mbar_init(bar(BAR_B_EMPTY + i), 2); }
        for (int i = 0; i < kDBufs; i++) { mbar_init(bar(BAR_D_FULL + i), 1); mbar_init(bar(BAR_D_EMPTY + i), 8); }
        mbar_init(bar(BAR_END), 1); mbar_init(bar(BAR_END + 1), 1);
        for (int i = 0; i < 8; i++) { mbar_init(bar(BAR_A_FULL + i), 8); mbar_init(bar(BAR_A_EMPTY + i), 1); }
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 17) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&s_tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    volatile int *abortp = &s_abort;
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");

    const int G = g.G, nreal = (G + kChunk - 1) / kChunk, nchunks = nreal + g.pseudo;
    // The units left for a last, partly filled wave are cut into their tiles where every tile then gets an SM of its own; a tile by
    // itself takes 0.6 (20 tokens) to 0.8 (96) of the two's time.  Measured, 4096 inputs, whole then cut: 17408 rows, 20 tokens 39
    // and 27 us, 96 tokens 50 and 45; 28608 rows, 300 tokens (3 waves and 4 units) 133 and 119; more units than half of the SMs are
    // left whole, since the tiles would take two turns.  The counts stay in shared memory: registers are short, and a unit is long.
    // (Not for the experts: what it adds to a unit cost more there, units being short, than the last wave of many gives.)
    const int all = (MODE == kProj ? (g.p.n + kTok - 1) / kTok : uniform(*g.p.plan.njobs)) * g.units_per_job;
    if (MODE == kProj) {
        if (tid == 0) {
            const int rest = all % (int)gridDim.x;
            const bool cut = 2 * rest <= (int)gridDim.x;
            s_whole = cut ? all - rest : all;
            s_units = cut ? all + rest : all;
        }
        __syncthreads();
    }
    auto units = [&]() { return MODE == kProj ? *(volatile int *)&s_units : all; };
    auto whole = [&]() { return MODE == kProj ? *(volatile int *)&s_whole : all; };
    const size_t s_pitch = (size_t)G * 2;
    // after a wait that ran out: the copies in flight land before the CTA goes (a ring's last `count` loads)
    auto drain = [&](int first, int n, int slot, uint32_t phase, int count) {
        const long long t0 = clock64();
        for (int i = 0; i < count; i++) {
            if (slot == 0) { slot = n; phase ^= 1; }
            slot--;
            while (!mbar_try(bar(first + slot), phase) && clock64() - t0 < 200000000LL) {}
        }
    };
    // one thread's row of a tile: its scales and biases (rows beyond the matrix read the last one; their results are dropped)
    auto row_ptr = [&](const Unit &u, int tile, int r, bool biases) {
        const Q4View &m = g.p.mat[tile_mat<MODE>(u, tile)];
        const int first = tile_row<MODE>(u, tile);
        const unsigned char *tile0 = (biases ? m.biases : m.scales) + (size_t)u.expert * m.s_stride + (size_t)first * s_pitch;  // uniform
        return tile0 + (uint32_t)min(r, m.rows - 1 - first) * (uint32_t)s_pitch;
    };

    auto matrix_bytes = [&](const Unit &u, int tile, bool biases) {
        const Q4View &m = g.p.mat[tile_mat<MODE>(u, tile)];
        const unsigned char *first = (biases ? m.biases : m.scales) + (size_t)u.expert * m.s_stride;
        return Bytes{first, first + (size_t)m.rows * s_pitch};
    };

    if (warp == 16) {
        // ================= TMA producer: tokens =================
        Ring<kBSlots> rb;
        int count = 0;
        bool ok = true;
        for (int u = blockIdx.x; u < units() && ok; u += gridDim.x) {
            const Unit un = unit_at<MODE>(g, u, whole());
            if (MODE == kProj && un.tiles == 0) break;
            for (int c = 0; c < nchunks && ok; c++) {
                const int first = c < nreal ? c * kChunk : G + c - nreal, ng = c < nreal ? min(kChunk, G - first) : 1;  // 64 columns of x each
                for (int j = 0; j < ng && ok; j += 2) {
                    ok = __all_sync(0xffffffffu, count < kBSlots || bar_wait(bar(BAR_B_EMPTY + rb.slot), rb.phase ^ 1, abortp));
                    if (!ok) break;
                    const uint32_t full = bar(BAR_B_FULL + rb.slot), dst = sB + (uint32_t)rb.slot * kBSlot + (uint32_t)lane * 2048u;
                    const int n = min(2, ng - j);
                    if (lane == 0) mbar_expect_tx(full, (uint32_t)(un.ncols * 256 * n));
                    __syncwarp();
                    if (lane * 16 < un.ncols)
                        for (int q = 0; q < n; q++) {
                            tma_load_2d(dst + (uint32_t)(2 * q) * kBTile, &maps.x, (first + j + q) * 64, un.start + lane * 16, full);
                            tma_load_2d(dst + (uint32_t)(2 * q + 1) * kBTile, &maps.x, g.kp + (first + j + q) * 64, un.start + lane * 16, full);
                        }
                    rb.next(); count = min(count + 1, kBSlots);
                }
            }
        }
        if (lane == 0 && *abortp) drain(BAR_B_FULL, kBSlots, rb.slot, rb.phase, count);
    } else if (warp == 18) {
        // ================= TMA producer: weights =================
        if (lane == 0) {
            Ring<kWSlots> rw;
            int count = 0;
            bool ok = true;
            for (int u = blockIdx.x; u < units() && ok; u += gridDim.x) {
                const Unit un = unit_at<MODE, false>(g, u, whole());
                if (MODE == kProj && un.tiles == 0) break;
                for (int c = 0; c < nchunks && ok; c++)
                    for (int i = 0; i < un.tiles && ok; i++) {
                        auto load = [&](const CUtensorMap *map, int x) {  // 128 bytes of each of the tile's rows
                            ok = count < kWSlots || bar_wait(bar(BAR_W_EMPTY + rw.slot), rw.phase ^ 1, abortp);
                            if (!ok) return;
                            mbar_expect_tx(bar(BAR_W_FULL + rw.slot), kWSlot);
                            tma_load_3d(sW + (uint32_t)rw.slot * kWSlot, map, x, tile_row<MODE>(un, i), un.expert, bar(BAR_W_FULL + rw.slot));
                            rw.next(); count = min(count + 1, kWSlots);
                        };
                        const int m = tile_mat<MODE>(un, i);
                        if (c < nreal) load(&maps.w[m], c * 32);
                        else if (WIDE) {
                            load(&maps.s[m], (c - nreal) * 64);
                            if (ok) load(&maps.b[m], (c - nreal) * 64);
                        }
                    }
            }
            if (*abortp) drain(BAR_W_FULL, kWSlots, rw.slot, rw.phase, count);
        }
        __syncwarp();
    } else if (warp == 17 || warp == 19) {
        // ================= MMA issuers =================
        // A warp per tile: while one waits and counts, the other's MMAs keep the tensor core busy (its queue holds two or three).
        // A whole warp walks the steps and one elected lane issues a slot's MMAs in one go: everything they read is then uniform
        // across the warp (the reductions say so to the compiler), and an MMA costs what the tensor core takes, 57 cycles at
        // N = 96.  Issued by `lane == 0` in divergent code each took 120 to 190.
        const int tile = warp == 17 ? 0 : 1;
        const uint32_t d = uniform(tmem) + kColStep + (uint32_t)(tile * kTok), a0 = uniform(tmem) + kColA;
        const uint64_t desc0 = smem_desc(sB, 0, 1024);
        constexpr uint64_t kTile = kBTile >> 4;  // in the descriptor's units of 16 bytes
        Ring<kBSlots> rb;
        // operand slots filled before this chunk (both tiles), of this tile (a pair of barriers of its own announces them, so that a
        // warp never waits on a phase it is two behind), steps of this tile
        uint32_t pairs = 0, mine = 0, steps = 0;
        bool ok = true;
        for (int u = blockIdx.x; u < units() && ok; u += gridDim.x) {
            const Unit un = unit_at<MODE>(g, u, whole());
            if (MODE == kProj && un.tiles == 0) break;
            const uint32_t idesc = idesc_dense(128, un.ncols, false, 0);
            for (int c = 0; c < nchunks && ok; c++) {
                const bool real = c < nreal;
                const int na = real ? min(kChunk, G - c * kChunk) : 2, npairs = (na + 1) / 2;
                const int nk = real ? 4 : (min(64, G - (c - nreal) * 64) + 15) / 16;  // the bias block: one column per group
                if (tile < un.tiles) {
                    uint32_t n = pairs + (uint32_t)(tile * npairs);
                    ok = steps == 0 || __all_sync(0xffffffffu, bar_wait(bar(BAR_D_EMPTY + tile), (steps - 1) & 1, abortp));
                    for (int q = 0; q < npairs && ok; q++, n++, mine++) {
                        const uint32_t slot = n % kA;
                        ok = __all_sync(0xffffffffu, bar_wait(bar(BAR_B_FULL + rb.slot), rb.phase, abortp) &&
                                                         bar_wait(bar(BAR_A_FULL + 2 * tile + (int)(mine & 1)), mine >> 1 & 1, abortp));
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t a = a0 + slot * 64;
                        const uint64_t b0 = desc0 + (uint64_t)(rb.slot * (kBSlot >> 4));
                        const bool two = 2 * q + 1 < na;
                        if (elect_one()) {
                            if (real) {
#pragma unroll
                                for (int k = 0; k < 4; k++) tc_mma_f16_ta(d, a + k * 8, b0 + kTile + k * 2, idesc, q > 0 || k > 0);  // lo
#pragma unroll
                                for (int k = 0; k < 4; k++) tc_mma_f16_ta(d, a + k * 8, b0 + k * 2, idesc, 1);  // hi
                                if (two) {
#pragma unroll
                                    for (int k = 0; k < 4; k++) tc_mma_f16_ta(d, a + 32 + k * 8, b0 + 3 * kTile + k * 2, idesc, 1);
#pragma unroll
                                    for (int k = 0; k < 4; k++) tc_mma_f16_ta(d, a + 32 + k * 8, b0 + 2 * kTile + k * 2, idesc, 1);
                                }
                            } else {
                                for (int k = 0; k < nk; k++) {
                                    tc_mma_f16_ta(d, a + k * 8, b0 + kTile + k * 2, idesc, k > 0);
                                    tc_mma_f16_ta(d, a + k * 8, b0 + k * 2, idesc, 1);
                                    tc_mma_f16_ta(d, a + 32 + k * 8, b0 + kTile + k * 2, idesc, 1);
                                    tc_mma_f16_ta(d, a + 32 + k * 8, b0 + k * 2, idesc, 1);
                                }
                            }
                            tc_commit(bar(BAR_A_EMPTY + slot));
                            tc_commit(bar(BAR_B_EMPTY + rb.slot));  // (the other warp's arrival and this one's free the token tile)
                            if (q == npairs - 1) tc_commit(bar(BAR_D_FULL + tile));
                        }
                        __syncwarp();
                        rb.next();
                    }
                    steps++;
                } else {
                    for (int q = 0; q < npairs && ok; q++) {  // no such tile in this unit: it only lets the token tiles go
                        ok = __all_sync(0xffffffffu, bar_wait(bar(BAR_B_FULL + rb.slot), rb.phase, abortp));
                        if (ok && lane == 0) mbar_arrive(bar(BAR_B_EMPTY + rb.slot));
                        rb.next();
                    }
                }
                pairs += (uint32_t)(un.tiles * npairs);
            }
        }
        if (!ok && elect_one()) {  // a wait ran out: let what was issued finish before tensor memory is given back
            tc_commit(bar(BAR_END + tile));
            const long long t0 = clock64();
            while (!mbar_try(bar(BAR_END + tile), 0) && clock64() - t0 < 200000000LL) {}
        }
        __syncwarp();
    } else if (warp < 8) {
        // ================= widen: weight tiles -> operand A =================
        const int wg = warp >> 2, r = (warp & 3) * 32 + lane;
        const uint32_t put_at = tmem + ((uint32_t)(warp & 3) << 21) + kColA + (uint32_t)(wg * 32);  // TMEM lane of the warp's first row in bits 16+
        // the row's words in a weight tile: this warp group's two groups of a chunk, 16-byte pieces swizzled by the row
        // (the second group four pieces on: bit 2 of the piece's number)
        const uint32_t piece0 = (uint32_t)r * 128u + (uint32_t)(((2 * wg) ^ (r & 7)) << 4), piece1 = (uint32_t)r * 128u + (uint32_t)(((2 * wg + 1) ^ (r & 7)) << 4);
        Ring<kWSlots> rw;
        Ring<kA> ra;
        Ring<kFSteps> rf;
        int ahead = 0;  // operand slots used so far (up to all); the two groups of four warps take a group of 64 inputs each
        bool ok = true;
        // one group's operand into its half of the next slot of TMEM
        uint32_t turn = 0;  // bit i: which of tile i's two barriers announces its next slot
        auto put = [&](const uint32_t (&a)[32], int i) {
            ok = __all_sync(0xffffffffu, ahead < kA || bar_wait(bar(BAR_A_EMPTY + ra.slot), ra.phase ^ 1, abortp));
            if (!ok) return;
            tc_fence_after();
            tc_st32(put_at + (uint32_t)(ra.slot * 64), a);
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(BAR_A_FULL + 2 * i + (int)(turn >> i & 1)));
            turn ^= 1u << i;
            ra.next();
            ahead = min(ahead + 1, kA);
        };
        // scales of the next chunk, a tile's row each: fetched a chunk ahead, those of a unit's first one before the bias block
        const unsigned char *sp[T];
        uint2 sc[T], sd[T];  // (not wide: two windows that hold the scales)
        auto window = [&](const Unit &un, int i, int c) { return window8((const unsigned char *)((uintptr_t)sp[i] & ~(uintptr_t)7) + 8 * c, matrix_bytes(un, i, false)); };
        auto aim = [&](const Unit &un) {
#pragma unroll
            for (int i = 0; i < T; i++) {
                const int t = i < un.tiles ? i : 0;
                sp[i] = row_ptr(un, t, r, false);
                if (WIDE) sc[i] = chunk_scales(sp[i], 0);
                else {
                    sc[i] = window(un, t, 0);
                    sd[i] = window(un, t, 1);
                }
            }
        };
        Unit un;
        int u = blockIdx.x;
        if (u < units()) {
            un = unit_at<MODE>(g, u, whole());
            if (MODE == kProj && un.tiles == 0) u = units();
            else aim(un);
        }
        while (u < units() && ok) {
            for (int c = 0; c < nreal && ok; c++) {
                const int na = min(kChunk, G - c * kChunk);
#pragma unroll 1  // (one copy of the loop's body: the four roles' code has to fit the instruction cache)
                for (int i = 0; i < un.tiles && ok; i++) {
                    uint2 s = i ? sc[1] : sc[0];
                    if (!WIDE) s = cut8(s, i ? sd[1] : sd[0], (uint32_t)(uintptr_t)(i ? sp[1] : sp[0]) & 7u, na);
                    if (c + 1 < nreal) {  // (in place: a copy of the result would wait for it)
                        if (WIDE) {
                            if (i) sc[1] = chunk_scales(sp[1], c + 1);
                            else sc[0] = chunk_scales(sp[0], c + 1);
                        } else if (i) {
                            sc[1] = sd[1];
                            sd[1] = window(un, 1, c + 2);
                        } else {
                            sc[0] = sd[0];
                            sd[0] = window(un, 0, c + 2);
                        }
                    }
                    bool far;
                    const int e = chunk_exponent(s, &far);
                    far = __any_sync(0xffffffffu, far);  // (both groups of warps see the scales of the same rows, so they agree)
                    const float up = pow2(127 + 141 - e);  // the largest scale comes to [2^14, 2^15)
                    // for the epilogue: what the step's sums have to be multiplied with (seen through A_FULL, the MMAs and D_FULL)
                    if (wg == 0) s_f[rf.slot * 128 + r] = pow2(127 + e - 141 + (far ? 8 : 24));
                    ok = __all_sync(0xffffffffu, bar_wait(bar(BAR_W_FULL + rw.slot), rw.phase, abortp));
                    if (!ok) break;
                    const uint32_t tile = sW + (uint32_t)rw.slot * kWSlot;
                    const uint4 ws[2][2] = {{ld_shared16(tile + piece0), ld_shared16(tile + piece1)}, {ld_shared16(tile + (piece0 ^ 64u)), ld_shared16(tile + (piece1 ^ 64u))}};
#pragma unroll
                    for (int q = 0; q < 2; q++) {  // (of an odd number of groups the last slot's second half is zeros)
                        if (2 * q >= na || !ok) break;
                        const uint4 w0 = ws[q][0], w1 = ws[q][1];
                        const uint32_t bits = q ? s.y : s.x;
                        const float mf = __uint_as_float(wg ? bits & 0xffff0000u : bits << 16) * up;
                        const float mq = far ? 0x1p15f : mf;
                        const uint32_t m = dup_h2(mq), m16 = dup_h2(mq * 0.0625f), mc = dup_h2(mq * -0x1p-21f);
                        uint32_t a[32];
                        widen_word(w0.x, m, m16, mc, a);
                        widen_word(w0.y, m, m16, mc, a + 4);
                        widen_word(w0.z, m, m16, mc, a + 8);
                        widen_word(w0.w, m, m16, mc, a + 12);
                        widen_word(w1.x, m, m16, mc, a + 16);
                        widen_word(w1.y, m, m16, mc, a + 20);
                        widen_word(w1.z, m, m16, mc, a + 24);
                        widen_word(w1.w, m, m16, mc, a + 28);
                        if (far) {
                            const uint32_t mh = dup_h2(mf + mf);
#pragma unroll
                            for (int k = 0; k < 32; k++) a[k] = mul_h2(a[k], mh);
                        }
                        put(a, i);
                    }
                    if (lane == 0) mbar_arrive(bar(BAR_W_EMPTY + rw.slot));  // (the last put brought the warp together)
                    rw.next();
                    rf.next();
                }
            }
            const Unit cur = un;
            u += gridDim.x;
            if (u < units()) {
                un = unit_at<MODE>(g, u, whole());
                if (MODE == kProj && un.tiles == 0) u = units();
                else aim(un);
            }
            for (int c = 0; c < g.pseudo && ok; c++) {
                const int gn = min(64, G - c * 64);
                for (int i = 0; i < cur.tiles && ok; i++) {
                    // b + 8 s of the row's groups; warps 0-3 take the first fp16 term, the others the second
                    float v[64];
                    uint32_t pw[32];
                    if (WIDE) {  // both tiles came like weight tiles, 64 bf16 to a row
                        Ring<kWSlots> rs = rw;
                        ok = __all_sync(0xffffffffu, bar_wait(bar(BAR_W_FULL + rs.slot), rs.phase, abortp));
                        const uint32_t srow = sW + (uint32_t)rs.slot * kWSlot + (uint32_t)r * 128u;
                        rs.next();
                        ok = ok && __all_sync(0xffffffffu, bar_wait(bar(BAR_W_FULL + rs.slot), rs.phase, abortp));
                        const uint32_t brow = sW + (uint32_t)rs.slot * kWSlot + (uint32_t)r * 128u;
                        if (!ok) break;
#pragma unroll
                        for (int q = 0; q < 8; q++) {
                            if (q * 8 >= gn) {
#pragma unroll
                                for (int k = 0; k < 8; k++) v[8 * q + k] = 0.f;
                                continue;
                            }
                            const uint4 s4 = ld_shared16(srow + (uint32_t)((q ^ (r & 7)) << 4)), b4 = ld_shared16(brow + (uint32_t)((q ^ (r & 7)) << 4));
                            const uint32_t sw[4] = {s4.x, s4.y, s4.z, s4.w}, bw[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                v[8 * q + 2 * k] = fmaf(8.f, __uint_as_float(sw[k] << 16), __uint_as_float(bw[k] << 16));
                                v[8 * q + 2 * k + 1] = fmaf(8.f, __uint_as_float(sw[k] & 0xffff0000u), __uint_as_float(bw[k] & 0xffff0000u));
                            }
                        }
                    } else {
                        const unsigned char *ps = row_ptr(cur, i, r, false) + c * 128, *pb = row_ptr(cur, i, r, true) + c * 128;
                        const unsigned char *ws = (const unsigned char *)((uintptr_t)ps & ~(uintptr_t)15), *wb = (const unsigned char *)((uintptr_t)pb & ~(uintptr_t)15);
                        const uint32_t os = (uint32_t)(ps - ws), ob = (uint32_t)(pb - wb);
                        const int ns = (int)(os + 2 * gn + 15) >> 4, nb = (int)(ob + 2 * gn + 15) >> 4;  // windows, at most 9
                        const Bytes ms = matrix_bytes(cur, i, false), mb = matrix_bytes(cur, i, true);
                        if (ws >= ms.begin && ws + 16 * ns <= ms.end && wb >= mb.begin && wb + 16 * nb <= mb.end) {
#pragma unroll
                            for (int h = 0; h < 2; h++) {  // 32 groups at a time: ten loads on their way together
                                uint4 s4[5], b4[5];
#pragma unroll
                                for (int q = 0; q < 5; q++) {
                                    s4[q] = 4 * h + q < ns ? window16(ws + 16 * (4 * h + q)) : make_uint4(0, 0, 0, 0);
                                    b4[q] = 4 * h + q < nb ? window16(wb + 16 * (4 * h + q)) : make_uint4(0, 0, 0, 0);
                                }
#pragma unroll
                                for (int q = 0; q < 4; q++) {
                                    const uint4 s8 = cut16(s4[q], s4[q + 1], os), b8 = cut16(b4[q], b4[q + 1], ob);
                                    const uint32_t sw[4] = {s8.x, s8.y, s8.z, s8.w}, bw[4] = {b8.x, b8.y, b8.z, b8.w};
#pragma unroll
                                    for (int k = 0; k < 4; k++) {
                                        const int at = 32 * h + 8 * q + 2 * k;
                                        v[at] = at < gn ? fmaf(8.f, __uint_as_float(sw[k] << 16), __uint_as_float(bw[k] << 16)) : 0.f;
                                        v[at + 1] = at + 1 < gn ? fmaf(8.f, __uint_as_float(sw[k] & 0xffff0000u), __uint_as_float(bw[k] & 0xffff0000u)) : 0.f;
                                    }
                                }
                            }
                        } else {  // a row at the matrix's edge
                            const uint16_t *hs = reinterpret_cast<const uint16_t *>(ps), *hb = reinterpret_cast<const uint16_t *>(pb);
#pragma unroll
                            for (int q = 0; q < 64; q++) v[q] = q < gn ? fmaf(8.f, bf16_bits_to_float(__ldg(hs + q)), bf16_bits_to_float(__ldg(hb + q))) : 0.f;
                        }
                    }
                    float m = 0.f;
#pragma unroll
                    for (int q = 0; q < 64; q++) m = fmaxf(m, fabsf(v[q]));
                    const int e = max((int)(__float_as_uint(m) >> 23), 16);
                    const float up = pow2(127 + 141 - e);  // the largest comes to [2^14, 2^15): as far up as fp16 goes
#pragma unroll
                    for (int q = 0; q < 32; q++) {
                        const float a0 = v[2 * q] * up, a1 = v[2 * q + 1] * up;
                        const __half2 h = __floats2half2_rn(a0, a1);
                        const float2 hf = __half22float2(h);
                        pw[q] = h2_bits(wg == 0 ? h : __floats2half2_rn(a0 - hf.x, a1 - hf.y));
                    }
                    if (wg == 0) s_f[rf.slot * 128 + r] = pow2(127 + e - 141) / kSumScale;
                    put(pw, i);
                    for (int k = 0; k < (WIDE ? 2 : 0); k++) {
                        if (lane == 0) mbar_arrive(bar(BAR_W_EMPTY + rw.slot));
                        rw.next();
                    }
                    rf.next();
                }
            }
        }
    } else {
        // ================= epilogue =================
        const int r = (warp & 3) * 32 + lane, half = (warp - 8) >> 2;  // columns half * 48 .. + 47
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;
        uint32_t seen = 0;  // bit i: parity of tile i's next step
        Ring<kFSteps> rf;
        bool ok = true;
        for (int u = blockIdx.x; u < units() && ok; u += gridDim.x) {
            const Unit un = unit_at<MODE>(g, u, whole());
            if (MODE == kProj && un.tiles == 0) break;
            // columns half * 48 + 32 q + lane: the row of the output it goes to, and what takes its token's power of two off again
            int out_row[2] = {0, 0};
            float ts[2] = {0.f, 0.f};
#pragma unroll
            for (int q = 0; q < 2; q++) {
                const int col = half * kHalf + q * 32 + lane;
                if (col >= un.cnt || q * 32 + lane >= kHalf) continue;
                out_row[q] = MODE == kDown ? g.p.plan.pair_of[un.start + col] : un.start + col;
                ts[q] = __ldg(g.tscale + un.start + col);
            }
            const int live = un.cnt - half * kHalf;  // columns of this warp that are tokens
            for (int c = 0; c < nchunks && ok; c++) {
                const bool last = c == nchunks - 1;
                for (int i = 0; i < un.tiles && ok; i++) {
                    ok = __all_sync(0xffffffffu, bar_wait(bar(BAR_D_FULL + i), seen >> i & 1, abortp));
                    if (!ok) break;
                    tc_fence_after();
                    uint32_t d[3][16];
                    const uint32_t tstep = tmem + lanes + kColStep + (uint32_t)(i * kTok + half * kHalf);
                    const uint32_t tsum = tmem + lanes + kColSum + (uint32_t)(i * kTok + half * kHalf);
                    if (live > 0) {
                        tc_ld16(tstep, d[0]);
                        if (live > 16) tc_ld16(tstep + 16, d[1]);
                        if (live > 32) tc_ld16(tstep + 32, d[2]);
                        tc_wait_ld();
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(BAR_D_EMPTY + i));
                    const float f = s_f[rf.slot * 128 + r];
                    rf.next();
                    seen ^= 1u << i;
                    uint64_t ff;
                    asm("mov.b64 %0, {%1, %1};\n" : "=l"(ff) : "f"(f));
                    const int row = tile_row<MODE>(un, i) + r;
                    float *out = g.p.out[MODE == kProj ? un.mat : 0] + row;
#pragma unroll
                    for (int q = 0; q < 3; q++) {  // 16 columns at a time
                        if (live <= q * 16) break;
                        uint32_t (&v)[16] = d[q], s[16];
                        if (c > 0) {
                            tc_ld16(tsum + q * 16, s);
                            tc_wait_ld();
#pragma unroll
                            for (int k = 0; k < 16; k += 2) fma_f32x2(v[k], v[k + 1], ff, s[k], s[k + 1]);
                        } else {
#pragma unroll
                            for (int k = 0; k < 16; k++) v[k] = __float_as_uint(__uint_as_float(v[k]) * f);
                        }
                        if (!last || (MODE == kGateUp && !(i & 1))) {
                            tc_st16(tsum + q * 16, v);
                            continue;
                        }
                        if constexpr (MODE == kGateUp) {  // the gate's sums wait one tile to the left
                            tc_ld16(tsum + q * 16 - kTok, s);
                            tc_wait_ld();
                        }
#pragma unroll
                        for (int k = 0; k < 16; k++) {
                            const int o = __shfl_sync(0xffffffffu, out_row[q >> 1], (q & 1) * 16 + k);
                            const float t = __shfl_sync(0xffffffffu, ts[q >> 1], (q & 1) * 16 + k);
                            float y = __uint_as_float(v[k]) * t;
                            if constexpr (MODE == kGateUp) {
                                const float a = __uint_as_float(s[k]) * t;
                                y = a / (1.f + expf(-a)) * y;
                            }
                            if (q * 16 + k < live && row < un.rows) out[(size_t)o * un.rows] = y;
                        }
                    }
                    tc_wait_st();
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 17) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512u) : "memory");
    }
    if (tid == 0 && s_abort) atomicExch(g.err, 0x60 + MODE);
}

// Rows of fp32 activations -> two fp16 terms each, brought into range by a power of two per row, in the order the widened
// words have along K (0 4 1 5 2 6 3 7 of every eight); behind them the sums of every 64 inputs, likewise in two terms.
// One CTA per row of the result; `source` (may be null): row i is row source[i] / per of x.
__global__ void __launch_bounds__(256)
q4_split_kernel(const float *__restrict__ x, int K, int kp, const int *count, const int *source, int per, __half *__restrict__ xs,
                float *__restrict__ tscale) {
    __shared__ float s_red[8], s_sum[8];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    const size_t row = blockIdx.x;
    if (count != nullptr && (int)row >= *count) return;
    const float4 *src = reinterpret_cast<const float4 *>(x + (source != nullptr ? (size_t)(source[row] / per) : row) * K);
    float am = 0.f, sum = 0.f;
    for (int i = tid; i < K / 4; i += 256) {
        const float4 v = __ldg(src + i);
        am = fmaxf(fmaxf(am, fmaxf(fabsf(v.x), fabsf(v.y))), fmaxf(fabsf(v.z), fabsf(v.w)));
        sum += (v.x - v.x) + (v.y - v.y) + (v.z - v.z) + (v.w - v.w);  // 0, or NaN where an input is not finite
    }
    am = warp_max(am);
    sum = warp_sum(sum);
    if (lane == 0) { s_red[warp] = am; s_sum[warp] = sum; }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; w++) { am = fmaxf(am, s_red[w]); sum += s_sum[w]; }
    const bool bad = !(sum == 0.f);
    // am in [2^e, 2^(e+1)) becomes [2^14, 2^15), as far up as fp16 goes, so that small inputs beside it keep their bits; the sums of
    // 64 inputs are stored 2^-6 times as large, which the widening warps make up for
    int e = max((int)(__float_as_uint(am) >> 23), 16);
    if (bad) e = 141;
    const float up = __uint_as_float((uint32_t)(127 + 141 - e) << 23);
    if (tid == 0) tscale[row] = bad ? __uint_as_float(0x7fc00000u) : __uint_as_float((uint32_t)(127 + e - 141) << 23);
    __half *hi = xs + row * 2 * kp, *lo = hi + kp;
    const int G = K / 64;
    for (int i0 = 0; i0 < K / 8; i0 += 256) {  // eight inputs per thread; the eight threads of a group are neighbours
        const int i = i0 + tid;
        const bool valid = i < K / 8;
        float v[8] = {};
        if (valid && !bad) {
            const float4 a = __ldg(src + 2 * i), b = __ldg(src + 2 * i + 1);
            v[0] = a.x * up; v[1] = a.y * up; v[2] = a.z * up; v[3] = a.w * up; v[4] = b.x * up; v[5] = b.y * up; v[6] = b.z * up; v[7] = b.w * up;
        }
        uint32_t h[4], l[4];
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const __half2 p = __floats2half2_rn(v[q], v[q + 4]);
            const float2 f = __half22float2(p);
            h[q] = h2_bits(p);
            l[q] = h2_bits(__floats2half2_rn(v[q] - f.x, v[q + 4] - f.y));
        }
        float s = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        s *= kSumScale;
        if (valid) {
            *reinterpret_cast<uint4 *>(hi + 8 * i) = make_uint4(h[0], h[1], h[2], h[3]);
            *reinterpret_cast<uint4 *>(lo + 8 * i) = make_uint4(l[0], l[1], l[2], l[3]);
            if ((i & 7) == 0) {
                const __half sh = __float2half_rn(s);
                hi[K + (i >> 3)] = sh;
                lo[K + (i >> 3)] = __float2half_rn(s - __half2float(sh));
            }
        }
    }
    for (int i = G + tid; i < kp - K; i += 256) { hi[K + i] = __float2half_rn(0.f); lo[K + i] = __float2half_rn(0.f); }
}

// [matrices][rows][row_bytes], box [1][128 rows][128 bytes], 128-byte swizzle, zeros outside
bool map_rows(CUtensorMap *m, const void *base, long long stride, int rows, int row_bytes, int matrices, bool words) {
    EncodeTiledFn enc = get_encode();
    if (!enc) return false;
    const cuuint32_t esz = words ? 4 : 2;
    const cuuint64_t dims[3] = {(cuuint64_t)row_bytes / esz, (cuuint64_t)rows, (cuuint64_t)matrices};
    const cuuint64_t strides[2] = {(cuuint64_t)row_bytes, (cuuint64_t)(matrices > 1 ? stride : (long long)rows * row_bytes)};
    const cuuint32_t box[3] = {128 / esz, 128, 1}, estr[3] = {1, 1, 1};
    return enc(m, words ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void *>(base), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <Q4Mode MODE, bool WIDE>
int launch_gemm(const GemmMaps &maps, GemmParams &g, long long jobs, int sm_count, cudaStream_t st) {
    constexpr int kRows = MODE == kGateUp ? T * 64 : T * 128;
    g.units_per_job = 0;
    for (int i = 0; i < (MODE == kProj ? g.p.nmat : 1); i++) {
        g.m_units[i] = (g.p.mat[i].rows + kRows - 1) / kRows;
        g.units_per_job += g.m_units[i];
    }
    static std::atomic<unsigned long long> configured{0};
    if (!raise_smem_limit(reinterpret_cast<const void *>(q4_gemm_kernel<MODE, WIDE>), kGemmSmem, &configured)) return -1;
    // (fewer units than SMs: as many CTAs as there are units or, cut, tiles; idle ones would crowd the others onto half of the GPU)
    const long long units = jobs * g.units_per_job;
    const int grid = (int)std::min<long long>(MODE == kProj && 2 * units <= sm_count ? 2 * units : units, sm_count);
    return launch_dependent(q4_gemm_kernel<MODE, WIDE>, dim3(grid), dim3(kGemmThreads), kGemmSmem, st, maps, g) == cudaSuccess ? 1 : -1;
}

}  // namespace

int q4_split_columns(int in_dim) { return in_dim + (in_dim / 64 + 63) / 64 * 64; }

int launch_q4_split(const float *x, int rows, int in_dim, const int *count, const int *source, int per, void *xs, float *tscale, cudaStream_t st) {
    return launch_dependent(q4_split_kernel, dim3(rows), dim3(256), 0, st, x, in_dim, q4_split_columns(in_dim), count, source, per,
                            reinterpret_cast<__half *>(xs), tscale) == cudaSuccess ? 1 : -1;
}

int launch_q4_gemm(Q4Mode mode, const Q4Params &p, const void *xs, int xs_rows, const float *tscale, int *err, int sm_count, cudaStream_t st) {
    GemmMaps maps;
    memset(&maps, 0, sizeof maps);
    GemmParams g = {};
    g.p = p; g.G = p.in_dim / 64; g.pseudo = (g.G + 63) / 64; g.kp = q4_split_columns(p.in_dim); g.tscale = tscale; g.err = err;
    const int matrices = mode == kProj ? 1 : p.num_experts;
    bool wide = g.G % 8 == 0;  // scales and biases then start on 16 bytes in every row
    for (int i = 0; i < p.nmat; i++) wide = wide && (((uintptr_t)p.mat[i].scales | (uintptr_t)p.mat[i].biases) & 15) == 0;
    for (int i = 0; i < p.nmat; i++) {
        const Q4View &m = p.mat[i];
        if (!map_rows(&maps.w[i], m.w, m.w_stride, m.rows, p.in_dim / 2, matrices, true)) return -1;
        if (wide && (!map_rows(&maps.s[i], m.scales, m.s_stride, m.rows, g.G * 2, matrices, false) ||
                       !map_rows(&maps.b[i], m.biases, m.s_stride, m.rows, g.G * 2, matrices, false)))
            return -1;
    }
    if (!make_map_2d(&maps.x, xs, (uint64_t)xs_rows, (uint64_t)2 * g.kp, 16, false)) return -1;
    const long long jobs = mode == kProj ? (p.n + kTok - 1) / kTok : (long long)p.n * p.top_k;
    if (mode == kProj) return wide ? launch_gemm<kProj, true>(maps, g, jobs, sm_count, st) : launch_gemm<kProj, false>(maps, g, jobs, sm_count, st);
    if (mode == kGateUp) return wide ? launch_gemm<kGateUp, true>(maps, g, jobs, sm_count, st) : launch_gemm<kGateUp, false>(maps, g, jobs, sm_count, st);
    return wide ? launch_gemm<kDown, true>(maps, g, jobs, sm_count, st) : launch_gemm<kDown, false>(maps, g, jobs, sm_count, st);
}

}  // namespace fm
