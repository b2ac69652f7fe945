// Products of 4-bit affine matrices with a few tokens each: projections at decode, and the routed experts while an
// expert sees a handful of tokens.
//
// Reference: cpu_dequant_matvec (metal_infer/cpu_kernels.h:199-232; Metal dequant_matvec_4bit*), batched over matrices
// that share their input by gpu_encode_batch_matvec (metal_infer/gpu_dispatch.h), and the experts' gate / up / SwiGLU /
// down chain of the same file.
//     y[r] = sum over groups g of 64 inputs:  s[r][g] * sum_k nibble[r][k] x[k]  +  b[r][g] * X[g],   X[g] = sum_k x[k]
//
// The weights' stream, 0.5625 bytes per weight, is what it cannot do without; next to it stand the instructions that widen
// them.  So the nibbles are never turned into floating point: they are multiplied as they are, unsigned bytes, on the integer
// tensor cores (mma.sync m16n8k32, measured at twice the fp16 rate), which takes 3 instructions per word of eight.  The
// activations are the other factor, as 32-bit fixed point relative to the largest of their group of 64, cut into four
// signed bytes, which are four of the eight columns of the product.  The other four are a second token; or, for one token,
// a second group, so that a row is read 64 bytes at a time and not 32.  The integer sums are exact; what is left of fp32's
// accuracy is 2^-30 of a group's largest input.  Scale and bias meet the group's sum in fp32, once per row and group.
//
// A unit is 32 rows (kGateUp: 16 of gate and the same 16 of up) per warp along the rows, for one job.  The 8 warps of a CTA
// split the steps of a row (four groups each) and the unit's rows among themselves, by a cost rule in launch_one, and meet in
// shared memory at the unit's end; a lane fetches its words straight into registers, and refills them as it unpacks them, so
// that about 60 KB per SM are under way.  CTAs are persistent and take a contiguous range of units, so that a job's
// activations are widened once per CTA and not once per unit, and the next unit's weights are fetched while this one's sums
// meet.
//
// Measured (B200, as replayed graphs): one token x 4096 x 17408 in 11 us (40 MB: 3.6 TB/s; 5.3 TB/s in the long run, 4.5 us go into
// the start and the end), x 8192 x 4096 in 9 us; one token through 10 of 512 experts of 4096 x 1024 in 28 us with the weighted sum; 48
// tokens through them (2.2 GB) in 450 us, 4.9 TB/s.  Calls on fresh inputs take 14.5, 32 and 480 us.  In the long run it is bound by the L1 cache's wavefronts (72 % of their peak): a
// request of a warp touches 8 rows, 64 or 32 bytes of each, and the scales and biases cost as many as the words.
// One token in the two-token form: 12.5 and 35 us; the one-token form for 3 or more tokens takes 1.3 to 1.8 times as long.
// Rows read 64 bytes at a time for more tokens too, a group's share of the columns zero in the lanes of the other, doubles the
// products: 5 % faster at 2 tokens, 1.2 to 1.4 times as long from 4 on.
#include <math.h>

#include <algorithm>

#include "fm_device.cuh"
#include "fm_internal.h"

namespace fm {

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kTiles = 2;        // 16-row tiles per unit
constexpr int kTokBytes = 256;   // a token's group as bytes: 64 inputs x 4
// What the running sums count: 2^16, so that inputs up to fp32's largest number do not take a group's sums beyond it, where its
// scale is that of a weight.  (Sums below fp32's normal numbers are exact multiples of 2^-149 * 2^16 until a scale meets them.)
constexpr float kUnit = 65536.f;
constexpr int kFactorBytes = 32; // (factor, input sum) for each of the four lanes of a quad: per group and pair of tokens, or per two groups

__device__ __forceinline__ void mma_u8s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// the same with nothing to add to
__device__ __forceinline__ void mma_u8s8_first(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
}

// Eight inputs (those of one weight word, number wi of the group's) of a token -> fixed point bytes in the order of the B
// fragments, digit planes kPlane bytes apart.  The eight threads of a group of 64 inputs sit in consecutive lanes.
template <int kPlane>
__device__ __forceinline__ void widen8(const float4 &a, const float4 &b, bool valid, unsigned char *o, float2 *factor, int wi) {
    const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    float am = 0.f, sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) am = fmaxf(am, fabsf(v[i]));
    constexpr float u = 1.f / kUnit;
    sum = (fmaf(v[0], u, v[1] * u) + fmaf(v[2], u, v[3] * u)) + (fmaf(v[4], u, v[5] * u) + fmaf(v[6], u, v[7] * u));
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, o));
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    if (!valid) return;
    // am in [2^e, 2^(e+1)): inputs as integers of 2^(e-29), so that |q| < 2^30; groups below 2^-97 keep a fixed step.
    // A group with an infinity or a NaN (the maximum passes NaN by, the sum does not; of finite inputs it stays finite) makes its
    // token's results NaN.
    int e = (int)(__float_as_uint(am) >> 23) - 127;
    e = max(e, -97);
    const bool bad = !(fabsf(sum) <= 3.4028235e38f) || e > 127;
    const float up = __uint_as_float((uint32_t)(127 + 29 - e) << 23), down = bad ? __uint_as_float(0x7fc00000u) : __uint_as_float((uint32_t)(127 - 29 + e) << 23);
    uint32_t q[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int k = bad ? 0 : __float2int_rn(v[i] * up);
        // four signed digits of 8 bits: adding 0x80 to the lower three bytes carries into the next, flipping their top bit
        // takes it off again
        q[i] = ((uint32_t)k + 0x00808080u) ^ 0x00808080u;
    }
    // digit planes: plane p (0 = most significant) of the even inputs and of the odd ones
#pragma unroll
    for (int half = 0; half < 2; half++) {
        const uint32_t a = q[half], b = q[2 + half], c = q[4 + half], d = q[6 + half];
        const uint32_t ab_hi = __byte_perm(a, b, 0x7362), cd_hi = __byte_perm(c, d, 0x7362);  // a2 b2 a3 b3
        const uint32_t ab_lo = __byte_perm(a, b, 0x5140), cd_lo = __byte_perm(c, d, 0x5140);  // a0 b0 a1 b1
        *reinterpret_cast<uint32_t *>(o + 0 * kPlane + half * 4) = __byte_perm(ab_hi, cd_hi, 0x7632);  // a3 b3 c3 d3
        *reinterpret_cast<uint32_t *>(o + 1 * kPlane + half * 4) = __byte_perm(ab_hi, cd_hi, 0x5410);  // a2 b2 c2 d2
        *reinterpret_cast<uint32_t *>(o + 2 * kPlane + half * 4) = __byte_perm(ab_lo, cd_lo, 0x7632);  // a1 b1 c1 d1
        *reinterpret_cast<uint32_t *>(o + 3 * kPlane + half * 4) = __byte_perm(ab_lo, cd_lo, 0x5410);  // a0 b0 c0 d0
    }
    // the pair of upper digits counts 2^16, the pair of lower ones 1; the input sum goes with either (see the loop)
    if (wi < 2) factor[wi] = make_float2(wi == 0 ? down * (65536.f / kUnit) : down / kUnit, sum);
}

constexpr int S = 4;             // groups per step
// A step of a row pair as a lane holds it: 8 bytes of words per group and row, the scales of rows g and g + 8, and the bias of
// row g (even lanes) or g + 8 (odd lanes).
template <bool ONE>
struct Held {
    uint2 w[kTiles][2][S];
    uint2 sc[kTiles][2], bi[kTiles];
};
// One token: 16 bytes of words per two groups and row.  Lanes 0 and 1 of a quad hold the first group, 2 and 3 the second.
template <>
struct Held<true> {
    uint4 w[kTiles][2][S / 2];
    uint2 sc[kTiles][2], bi[kTiles];
};
// The bf16 numbers of a step's groups: in one read where a row of them is a multiple of 8 bytes, 8-byte aligned; else one by
// one, those behind the row's end repeating its last (their activations count nothing).
template <bool WIDE>
__device__ __forceinline__ uint2 load_bf16s(const unsigned char *row, int step, int G) {
    if constexpr (WIDE) {
        return __ldg(reinterpret_cast<const uint2 *>(row) + step);
    } else {
        const uint16_t *p = reinterpret_cast<const uint16_t *>(row);
        const int j = step * S, last = G - 1;
        return make_uint2((uint32_t)__ldg(p + j) | (uint32_t)__ldg(p + min(j + 1, last)) << 16,
                          (uint32_t)__ldg(p + min(j + 2, last)) | (uint32_t)__ldg(p + min(j + 3, last)) << 16);
    }
}
__device__ __forceinline__ float bf16_at(uint2 four, int j) {
    const uint32_t pair = j & 2 ? four.y : four.x;
    return __uint_as_float(j & 1 ? pair & 0xffff0000u : pair << 16);
}
// of two groups' bf16 numbers that of the lane's (up: 16 for the first group, 0 for the second)
__device__ __forceinline__ float bf16_of(uint32_t pair, int up) { return __uint_as_float((pair << up) & 0xffff0000u); }
// The same value in every lane, and known to the compiler as such (values of at least 0).
__device__ __forceinline__ int uniform(int v) { return __reduce_max_sync(0xffffffffu, v); }

// Warps: WK of them side by side along a row's steps, 8 / WK along the rows.
template <Q4Mode MODE, int NTL, bool WIDE>
__global__ void __launch_bounds__(kThreads, NTL == 4 ? 1 : 2)
q4_stream_kernel(const __grid_constant__ Q4Params p, int chunk_groups, int units_per_job, int fixed_jobs, int wk_log2, int sms) {
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr bool ONE = NTL == 0;
    constexpr int kTok = ONE ? 1 : 2 * NTL, NT = ONE ? 1 : NTL;
    constexpr int kAhead = NTL == 4 ? 4 : 1;  // words of activations a thread has under way: as many as fit beside the weights' registers
    unsigned char *s_b = smem;                                                                      // [tokens][chunk][256]
    float2 *s_f = reinterpret_cast<float2 *>(smem + (size_t)kTok * chunk_groups * kTokBytes);       // [NT][chunk][4], or [chunk / 2][4]
    float *s_red = reinterpret_cast<float *>(reinterpret_cast<unsigned char *>(s_f) + (size_t)NT * chunk_groups * kFactorBytes);  // [2][warp][tok][32 rows]
    const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int WK = 1 << wk_log2, wk = warp & (WK - 1), wr = warp >> wk_log2, rows_unit = (MODE == kGateUp ? 16 : 32) * (kWarps >> wk_log2);
    const int G = p.in_dim / 64;
    const uint32_t w_pitch = (uint32_t)G * 32, s_pitch = (uint32_t)G * 2;
    const int nchunks = (G + chunk_groups - 1) / chunk_groups;
    // The weights, the ids and the plan were there before the gate / up launch in front of a kDown one began (that one waited for
    // them): only its activations have to be waited for, so the first weights are fetched under its tail.
    if constexpr (MODE != kDown) asm volatile("griddepcontrol.wait;\n" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    const int njobs = p.plan.njobs != nullptr ? uniform(*p.plan.njobs) : fixed_jobs;
    const long long units = (long long)njobs * units_per_job;
    // Ranges differ by a unit; those of the CTAs that share an SM (b, b + sms) are neighbours, so that no SM gets the longer ones only.
    const int range = gridDim.x % sms == 0 ? (int)(blockIdx.x % sms * (gridDim.x / sms) + blockIdx.x / sms) : (int)blockIdx.x;
    const long long u0 = units * range / gridDim.x, u1 = units * (range + 1) / gridDim.x;

    struct Unit {
        int job, expert, start, cnt, mat, row0;
    };
    auto pair_at = [&](int start, int i) { return MODE == kProj ? start + i : p.plan.njobs != nullptr ? p.plan.pair_of[start + i] : start; };
    auto enter_job = [&](Unit &r) {
        if constexpr (MODE == kProj) {
            r.expert = 0; r.start = r.job * kTok; r.cnt = min(kTok, p.n - r.start);
        } else if (r.job >= njobs) {
            r.cnt = 0;
        } else if (p.plan.njobs != nullptr) {
            const int4 j = p.plan.jobs[r.job];
            r.expert = uniform(j.x); r.start = uniform(j.y); r.cnt = uniform(j.z);
        } else {  // -1: a slot without an expert here
            r.expert = uniform(local_expert(p.ids[r.job], p.first_expert, p.num_experts) + 1) - 1;
            r.start = r.job; r.cnt = r.expert >= 0 ? 1 : 0;
        }
    };

    Held<ONE> h;
    // where the lane's rows start: offsets of rows g and g + 8 of each tile (rows without a place read the last one there is)
    const unsigned char *bw[kTiles], *bs[kTiles], *bb[kTiles];
    uint32_t ow[kTiles][2], os[kTiles][2], ob[kTiles];
    // where the rows of a unit start; the next unit of the same matrix, all of its rows in place, only moves the starts on
    bool whole = false;
    int at_job = -1, at_mat = -1;
    auto aim = [&](const Unit &un) {
        const bool fits = un.row0 + rows_unit <= p.mat[un.mat].rows;
        if (whole && fits && un.job == at_job && un.mat == at_mat) {
#pragma unroll
            for (int i = 0; i < kTiles; i++) {
                bw[i] += (size_t)rows_unit * w_pitch; bs[i] += (uint32_t)rows_unit * s_pitch; bb[i] += (uint32_t)rows_unit * s_pitch;
            }
            return;
        }
        whole = fits; at_job = un.job; at_mat = un.mat;
#pragma unroll
        for (int i = 0; i < kTiles; i++) {
            const Q4View &m = p.mat[MODE == kGateUp ? i : un.mat];
            const int want = un.row0 + (MODE == kGateUp ? 16 * wr : 32 * wr + 16 * i), first = min(want, m.rows - 1), last = m.rows - 1 - first;
            bw[i] = m.w + (size_t)un.expert * m.w_stride + (size_t)first * w_pitch;
            bs[i] = m.scales + (size_t)un.expert * m.s_stride + (size_t)first * s_pitch;
            bb[i] = m.biases + (size_t)un.expert * m.s_stride + (size_t)first * s_pitch;
            const uint32_t l0 = min(g, last), l1 = min(g + 8, last);
            ow[i][0] = l0 * w_pitch + t * (ONE ? 16 : 8); ow[i][1] = l1 * w_pitch + t * (ONE ? 16 : 8);
            os[i][0] = l0 * s_pitch; os[i][1] = l1 * s_pitch;
            ob[i] = t & 1 ? os[i][1] : os[i][0];
        }
    };
    const unsigned char *pw[kTiles][2];  // the step being fetched
    int left = S;                        // its groups that exist
    auto point = [&](int step) {
#pragma unroll
        for (int i = 0; i < kTiles; i++)
#pragma unroll
            for (int q = 0; q < 2; q++) pw[i][q] = bw[i] + (ow[i][q] + (uint32_t)step * (S * 32u));
        if constexpr (!WIDE) left = G - step * S;
    };
    auto fetch_words = [&](int j) {  // group j of the step; ONE: groups 2 j and 2 j + 1 (behind the row's end: its last group again)
        if constexpr (ONE) {
            const int at = WIDE ? j * 64 : j * 64 - 32 * max(0, 2 * j + (t >> 1) - (left - 1));
#pragma unroll
            for (int i = 0; i < kTiles; i++)
#pragma unroll
                for (int q = 0; q < 2; q++) h.w[i][q][j] = __ldg(reinterpret_cast<const uint4 *>(pw[i][q] + at));
        } else {
#pragma unroll
            for (int i = 0; i < kTiles; i++)
#pragma unroll
                for (int q = 0; q < 2; q++) h.w[i][q][j] = __ldg(reinterpret_cast<const uint2 *>(pw[i][q] + (WIDE ? j : min(j, left - 1)) * 32));
        }
    };
    auto fetch_scales = [&](int step) {
#pragma unroll
        for (int i = 0; i < kTiles; i++) {
            h.sc[i][0] = load_bf16s<WIDE>(bs[i] + os[i][0], step, G);
            h.sc[i][1] = load_bf16s<WIDE>(bs[i] + os[i][1], step, G);
            h.bi[i] = load_bf16s<WIDE>(bb[i] + ob[i], step, G);
        }
    };

    int held_start = -1, held_job = -1;  // whose activations shared memory holds
    int half = 0;                        // of s_red: units alternate
    auto next_unit = [&](long long &u, Unit &un) {  // the next one that has tokens
        do {
            if (++u >= u1) return;
            un.row0 += rows_unit;
            if (un.row0 >= p.mat[un.mat].rows) {
                un.row0 = 0;
                if (MODE == kProj && un.mat + 1 < p.nmat) {
                    un.mat++;
                } else {
                    un.mat = 0; un.job++;
                    enter_job(un);
                }
            }
        } while (un.cnt == 0);
    };
    long long u = u0;
    Unit un = {};
    un.job = (int)(u0 / units_per_job);
    {
        int rb = (int)(u0 - (long long)un.job * units_per_job);
        if constexpr (MODE == kProj)
            while (rb >= (p.mat[un.mat].rows + rows_unit - 1) / rows_unit) rb -= (p.mat[un.mat++].rows + rows_unit - 1) / rows_unit;
        un.row0 = rb * rows_unit;
        enter_job(un);
        if (u < u1 && un.cnt == 0) next_unit(u, un);
    }
    auto fetch_first = [&]() {
        point(wk);
#pragma unroll
        for (int j = 0; j < (ONE ? S / 2 : S); j++) fetch_words(j);
        fetch_scales(wk);
    };
    const bool has_first = wk < (min(chunk_groups, G) + S - 1) / S;  // this warp has a step in a unit's first chunk
    if (u < u1) {
        aim(un);
        if (has_first) fetch_first();
    }
    if constexpr (MODE == kDown) asm volatile("griddepcontrol.wait;\n" ::: "memory");
    // B fragments: two tokens -- column g is digit g & 3 of token g / 4 of the pair.  One token: column g is digit g & 3 of group g / 4
    // of two, and only the lanes that hold that group's words have anything in it; so a row is read 64 bytes at a time.
    const bool mine = (g >> 2) == (t >> 1);
    const int up = t < 2 ? 16 : 0;  // bf16_of: which of two scales is the lane's
    const unsigned char *lane_b = ONE ? s_b + (t * 4 + (g & 3)) * 32 : s_b + (size_t)(g >> 2) * chunk_groups * kTokBytes + ((g & 3) * 4 + t) * 16;
    while (u < u1) {
        const int ntl = (un.cnt + 1) / 2;
        float acc[kTiles][2][NT] = {}, accb[kTiles][NT] = {};
        Unit nx = un;
        long long v = u;
        for (int c = 0; c < nchunks; c++) {
            const int cg0 = c * chunk_groups, cgn = min(chunk_groups, G - cg0), step0 = cg0 / S, steps = (cgn + S - 1) / S;
            // activations of the job: of one token the source is the token, so consecutive single-token jobs share them
            int source = un.start;
            if (MODE == kGateUp && un.cnt == 1) source = pair_at(un.start, 0) / p.top_k;
            const int kind = MODE == kGateUp && un.cnt == 1 ? -2 : un.job;
            if (nchunks > 1 || kind != held_job || source != held_start) {
                __syncthreads();  // everyone is done with the previous activations
                const int words = cgn * 8, total = un.cnt * words;
                int tok = 0, w8 = tid;
                for (int i0 = 0; i0 < total; i0 += kAhead * kThreads) {  // the loads of a batch are under way before the first is used
                    float4 xa[kAhead], xb[kAhead];
                    int at[kAhead], who[kAhead];
#pragma unroll
                    for (int k = 0; k < kAhead; k++) {
                        while (w8 >= words && tok < un.cnt) { w8 -= words; tok++; }
                        at[k] = w8; who[k] = tok;
                        if (tok < un.cnt) {
                            int row = pair_at(un.start, tok);
                            if (MODE == kGateUp) row /= p.top_k;
                            const float4 *src = reinterpret_cast<const float4 *>(p.x + (size_t)row * p.in_dim + (size_t)cg0 * 64 + (size_t)w8 * 8);
                            xa[k] = __ldg(src); xb[k] = __ldg(src + 1);
                        } else {
                            xa[k] = xb[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                        }
                        w8 += kThreads;
                    }
#pragma unroll
                    for (int k = 0; k < kAhead; k++) {
                        const int grp = at[k] >> 3, wi = at[k] & 7;
                        if constexpr (ONE) {  // two groups' sixteen words in fours, a lane of the quad each
                            const int w = (grp & 1) * 8 + wi;
                            widen8<32>(xa[k], xb[k], who[k] < un.cnt, s_b + (size_t)(grp >> 1) * 2 * kTokBytes + (w >> 2) * 128 + (w & 3) * 8, s_f + (size_t)grp * 2, wi);
                        } else {
                            widen8<64>(xa[k], xb[k], who[k] < un.cnt, s_b + ((size_t)who[k] * chunk_groups + grp) * kTokBytes + (wi >> 1) * 16 + (wi & 1) * 8,
                                       s_f + ((size_t)(who[k] >> 1) * chunk_groups + grp) * 4 + (who[k] & 1) * 2, wi);
                        }
                    }
                }
                // the last step's groups behind the row's end count nothing
                constexpr int kPer = ONE ? 2 : 4;  // factors of a group
                for (int i = tid; i < NT * kPer * (steps * S - cgn); i += kThreads) {
                    const int nt = i / (kPer * (steps * S - cgn)), q = i - nt * kPer * (steps * S - cgn);
                    s_f[((size_t)nt * chunk_groups + cgn) * kPer + q] = make_float2(0.f, 0.f);
                }
                held_start = source; held_job = kind;
                __syncthreads();
            }
            for (int st = wk; st < steps; st += WK) {
                // what comes into the registers as this step leaves them: the warp's next step, of this chunk, of the next one, or of
                // the next unit
                int more = st + WK < steps ? step0 + st + WK : -1;
                if (more < 0) {
                    if (c + 1 < nchunks) {
                        if (wk < (min(chunk_groups, G - cg0 - chunk_groups) + S - 1) / S) more = step0 + steps + wk;
                    } else {
                        next_unit(v, nx);
                        if (v < u1) {
                            aim(nx);
                            if (has_first) more = wk;
                        }
                    }
                }
                uint2 sc[kTiles][2], bi[kTiles];
#pragma unroll
                for (int i = 0; i < kTiles; i++) { sc[i][0] = h.sc[i][0]; sc[i][1] = h.sc[i][1]; bi[i] = h.bi[i]; }
                if (more >= 0) { fetch_scales(more); point(more); }
                const unsigned char *fb = lane_b + (size_t)st * S * kTokBytes;
                const float2 *ff = s_f + (size_t)st * S * (ONE ? 2 : 4) + t;
                if constexpr (ONE) {
#pragma unroll
                    for (int b = 0; b < S / 2; b++) {
                        uint4 b01 = make_uint4(0, 0, 0, 0), b23 = b01;
                        if (mine) {
                            const uint4 *src = reinterpret_cast<const uint4 *>(fb + b * 2 * kTokBytes);
                            b01 = src[0]; b23 = src[1];
                        }
                        const float2 f = ff[b * 4];
                        uint32_t a[kTiles][4][4];  // nibbles as bytes: [tile][word of the lane's four][fragment register]
#pragma unroll
                        for (int i = 0; i < kTiles; i++) {
                            const uint4 w0 = h.w[i][0][b], w1 = h.w[i][1][b];
                            const uint32_t r0[4] = {w0.x, w0.y, w0.z, w0.w}, r1[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
                            for (int w = 0; w < 4; w++) {
                                a[i][w][0] = r0[w] & 0x0F0F0F0Fu; a[i][w][1] = r1[w] & 0x0F0F0F0Fu;
                                a[i][w][2] = (r0[w] >> 4) & 0x0F0F0F0Fu; a[i][w][3] = (r1[w] >> 4) & 0x0F0F0F0Fu;
                            }
                        }
                        if (more >= 0) fetch_words(b);
#pragma unroll
                        for (int i = 0; i < kTiles; i++) {
                            int d[4];
                            mma_u8s8_first(d, a[i][0][0], a[i][0][1], a[i][0][2], a[i][0][3], b01.x, b01.y);
                            mma_u8s8(d, a[i][1][0], a[i][1][1], a[i][1][2], a[i][1][3], b01.z, b01.w);
                            mma_u8s8(d, a[i][2][0], a[i][2][1], a[i][2][2], a[i][2][3], b23.x, b23.y);
                            mma_u8s8(d, a[i][3][0], a[i][3][1], a[i][3][2], a[i][3][3], b23.z, b23.w);
                            // |d| <= 64 * 15 * 128, so two digits still fit an int; lane t holds the digit pair t & 1 of group t / 2
                            // (the factor is a power of two and goes to the integer, exactly; a small one would leave a scale few bits)
                            acc[i][0][0] = fmaf(bf16_of(b ? sc[i][0].y : sc[i][0].x, up), f.x * (float)(d[0] * 256 + d[1]), acc[i][0][0]);
                            acc[i][1][0] = fmaf(bf16_of(b ? sc[i][1].y : sc[i][1].x, up), f.x * (float)(d[2] * 256 + d[3]), acc[i][1][0]);
                            accb[i][0] = fmaf(bf16_of(b ? bi[i].y : bi[i].x, up), f.y, accb[i][0]);
                        }
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < S; j++) {
                        uint32_t a[kTiles][2][4];  // nibbles as bytes: [tile][word of the lane's two][fragment register]
#pragma unroll
                        for (int i = 0; i < kTiles; i++) {
                            const uint2 w0 = h.w[i][0][j], w1 = h.w[i][1][j];
                            a[i][0][0] = w0.x & 0x0F0F0F0Fu; a[i][0][1] = w1.x & 0x0F0F0F0Fu;
                            a[i][0][2] = (w0.x >> 4) & 0x0F0F0F0Fu; a[i][0][3] = (w1.x >> 4) & 0x0F0F0F0Fu;
                            a[i][1][0] = w0.y & 0x0F0F0F0Fu; a[i][1][1] = w1.y & 0x0F0F0F0Fu;
                            a[i][1][2] = (w0.y >> 4) & 0x0F0F0F0Fu; a[i][1][3] = (w1.y >> 4) & 0x0F0F0F0Fu;
                        }
                        if (more >= 0) fetch_words(j);
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            if (nt >= ntl) break;
                            const uint4 bf = *reinterpret_cast<const uint4 *>(fb + (size_t)nt * 2 * chunk_groups * kTokBytes + j * kTokBytes);
                            const float2 f = ff[(size_t)nt * chunk_groups * 4 + j * 4];
#pragma unroll
                            for (int i = 0; i < kTiles; i++) {
                                int d[4];
                                mma_u8s8_first(d, a[i][0][0], a[i][0][1], a[i][0][2], a[i][0][3], bf.x, bf.y);
                                mma_u8s8(d, a[i][1][0], a[i][1][1], a[i][1][2], a[i][1][3], bf.z, bf.w);
                                // |d| <= 64 * 15 * 128, so two digits still fit an int; lane t holds the digit pair t & 1 of token t / 2
                                acc[i][0][nt] = fmaf(bf16_at(sc[i][0], j), f.x * (float)(d[0] * 256 + d[1]), acc[i][0][nt]);
                                acc[i][1][nt] = fmaf(bf16_at(sc[i][1], j), f.x * (float)(d[2] * 256 + d[3]), acc[i][1][nt]);
                                accb[i][nt] = fmaf(bf16_at(bi[i], j), f.y, accb[i][nt]);
                            }
                        }
                    }
                }
            }
        }
        if (v == u) {  // a warp without a step in the last chunk has not looked ahead yet
            next_unit(v, nx);
            if (v < u1) {
                aim(nx);
                if (has_first) fetch_first();
            }
        }
        // ---- the digit pairs of a row meet, then the warps along the row ----
        float *red = s_red + (size_t)half * kWarps * kTok * 32;
        half ^= 1;
#pragma unroll
        for (int i = 0; i < kTiles; i++)
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                float v0 = acc[i][0][nt] + (t & 1 ? 0.f : accb[i][nt]), v1 = acc[i][1][nt] + (t & 1 ? accb[i][nt] : 0.f);
                v0 += __shfl_xor_sync(0xffffffffu, v0, 1);
                v1 += __shfl_xor_sync(0xffffffffu, v1, 1);
                if constexpr (ONE) {  // and the two groups
                    v0 += __shfl_xor_sync(0xffffffffu, v0, 2);
                    v1 += __shfl_xor_sync(0xffffffffu, v1, 2);
                    if (t < 2) red[(size_t)warp * 32 + i * 16 + g + t * 8] = t ? v1 : v0;
                } else {
                    red[((size_t)warp * kTok + nt * 2 + (t >> 1)) * 32 + i * 16 + g + (t & 1) * 8] = t & 1 ? v1 : v0;
                }
            }
        __syncthreads();  // (the other half of s_red is free again once everyone is here)
        for (int e = warp; e < un.cnt * (kWarps >> wk_log2); e += kWarps) {  // 32 rows of one token per warp
            const int wq = e / un.cnt, tok = e - wq * un.cnt;
            float y = 0.f;
            for (int w = 0; w < WK; w++) y += red[((size_t)(wq * WK + w) * kTok + tok) * 32 + lane];
            y *= kUnit;
            const size_t pr = (size_t)pair_at(un.start, tok);
            const int row = un.row0 + (MODE == kGateUp ? wq * 16 : wq * 32) + lane;
            if constexpr (MODE == kGateUp) {
                const float up = __shfl_down_sync(0xffffffffu, y, 16);
                if (lane < 16 && row < p.mat[0].rows) p.out[0][pr * p.mat[0].rows + row] = y / (1.f + expf(-y)) * up;
            } else {
                if (row < p.mat[un.mat].rows) p.out[un.mat][pr * p.mat[un.mat].rows + row] = y;
            }
        }
        un = nx; u = v;
    }
}

constexpr int kMaxSmem = 200 * 1024;

size_t smem_bytes(int ntl, int chunk) {
    const int tokens = ntl == 0 ? 1 : 2 * ntl;
    return (size_t)tokens * chunk * kTokBytes + (size_t)std::max(1, ntl) * chunk * kFactorBytes + (size_t)2 * kWarps * tokens * 32 * 4;
}

template <Q4Mode MODE, int NTL, bool WIDE>
int launch_one(const Q4Params &p, int jobs, int sm_count, cudaStream_t st) {
    const int G = p.in_dim / 64;
    int chunk = (G + S - 1) / S * S;  // whole steps
    while (smem_bytes(NTL, chunk) > kMaxSmem) chunk = (chunk / 2 + S - 1) / S * S;
    const size_t smem = smem_bytes(NTL, chunk);
    static std::atomic<unsigned long long> configured{0};
    if (!raise_smem_limit(reinterpret_cast<const void *>(q4_stream_kernel<MODE, NTL, WIDE>), kMaxSmem, &configured)) return -1;
    const int grid_max = sm_count * std::max(1, std::min(NTL == 4 ? 1 : 2, (int)((220 * 1024) / (smem + 1024))));
    // Warps along a row, the others side by side on more rows.  An SM's time is its units' steps, plus a unit's end worth about
    // 0.6 of a step (the warps meet, the next unit's addresses), and it takes whole units: the cheapest split.  (One token x 4096
    // x 20480: 8, 4, 2 warps along a row take 16.7, 18.3 and 20.2 us; x 18944, where the last two come out even, 13.0, 12.7, 12.6.)
    int wk_log2 = 0, per_job = 0;
    double best = 0.0;
    for (int k = 0; k <= 3; k++) {
        const int rows = (MODE == kGateUp ? 16 : 32) * (kWarps >> k);
        int n = 0;
        for (int i = 0; i < (MODE == kGateUp ? 1 : p.nmat); i++) n += (p.mat[i].rows + rows - 1) / rows;
        const long long most = ((long long)jobs * n + sm_count - 1) / sm_count;
        const double cost = (double)most * ((double)(((G + S - 1) / S + (1 << k) - 1) >> k) + 0.6);
        if (k == 0 || cost < best) { best = cost; wk_log2 = k; per_job = n; }
    }
    const int grid = (int)std::min<long long>((long long)jobs * per_job, grid_max);
    return launch_dependent(q4_stream_kernel<MODE, NTL, WIDE>, dim3(grid), dim3(kThreads), smem, st, p, chunk, per_job, jobs, wk_log2, sm_count) == cudaSuccess ? 1 : -1;
}

template <Q4Mode MODE, int NTL>
int launch_steps(const Q4Params &p, int jobs, int sm_count, cudaStream_t st) {
    bool wide = p.in_dim % (64 * S) == 0;
    for (int i = 0; i < p.nmat; i++)
        wide = wide && (((uintptr_t)p.mat[i].scales | (uintptr_t)p.mat[i].biases | (uintptr_t)p.mat[i].s_stride) & 7) == 0;
    return wide ? launch_one<MODE, NTL, true>(p, jobs, sm_count, st) : launch_one<MODE, NTL, false>(p, jobs, sm_count, st);
}

}  // namespace

int launch_q4_stream(Q4Mode mode, const Q4Params &p, int sm_count, cudaStream_t st) {
    if (mode == kProj) {
        // tokens per pass over the weights: as many as there are, up to 8; more take more passes, which find the weights in L2
        if (p.n == 1) return launch_steps<kProj, 0>(p, 1, sm_count, st);
        if (p.n == 2) return launch_steps<kProj, 1>(p, 1, sm_count, st);
        if (p.n <= 4) return launch_steps<kProj, 2>(p, 1, sm_count, st);
        return launch_steps<kProj, 4>(p, (p.n + 7) / 8, sm_count, st);
    }
    const int pairs = p.n * p.top_k;  // an upper bound of the jobs; with a plan the device knows how many there are
    if (p.plan.njobs == nullptr) return mode == kGateUp ? launch_steps<kGateUp, 0>(p, pairs, sm_count, st) : launch_steps<kDown, 0>(p, pairs, sm_count, st);
    return mode == kGateUp ? launch_steps<kGateUp, 2>(p, pairs, sm_count, st) : launch_steps<kDown, 2>(p, pairs, sm_count, st);
}

}  // namespace fm
