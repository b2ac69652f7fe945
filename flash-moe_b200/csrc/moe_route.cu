// Routing of tokens to experts: scores, balance bias, groups, top-k, renormalised weights.
//
// Reference: cpu_softmax over the gate's logits, cpu_topk and the renormalisation of the selected weights between the
// post-attention norm and the experts of fused_layer_forward (metal_infer/layer_forward.h, metal_infer/cpu_kernels.h).
// Per token, over E logits x (include/fm_attn.h has the contract):
//     s_e = softmax(x)_e or 1 / (1 + exp(-x_e));   c_e = s_e + bias_e
//     groups: G runs of E / G experts; a group counts with the sum of its one or two best c; the best ones survive
//     ids = the top_k largest c, ties to the lowest index;   w = s, divided by the selected ones' sum, times a factor
//
// One warp per token, expert j * 32 + lane in register j: the row is read once, coalesced, and nothing leaves the
// registers.  Selection works on order-preserving 32-bit keys whose low bits make room for the expert's index, one redux
// per slot for value and holder together.  What bounds it is that chain (a redux and a pass over the lane's keys per slot),
// not the bytes: one token of 512 experts takes 4 us, all of it latency; 8192 tokens of 256 experts 8 us by softmax, 9.7 us by
// sigmoid, 11.8 us with a bias, 15.1 us with a bias and 8 groups (8.9 MB: the memory would take 1.4 us).
//
// Borders.  Which expert is the k-th best is a whole number, so a rounding must not decide it.  The chain therefore takes
// every expert that the lost bits, or the error of a 32-bit choice, leave possible -- one or two more than asked for -- and
// these few, one per lane, are put in their exact order wherever two neighbours leave a doubt: softmax without a
// bias by the logits themselves, sigmoid by choices in 64 bits.  Where that does not settle it (softmax with a bias, whose denominator would be needed in 64 bits;
// more than 32 candidates) the warp takes the whole row again in 64 bits; likewise the groups' totals, where two groups are
// at the border.
#include <math.h>

#include "fm_device.cuh"
#include "fm_internal.h"

namespace fm {

namespace {

constexpr int kRtWarps = 4;
constexpr unsigned kFull = 0xffffffffu;

// order-preserving map of non-NaN floats to unsigned; 0 is below every value (it stands for "not available")
__device__ __forceinline__ uint32_t key_of(float f) {
    const uint32_t u = __float_as_uint(f);
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k); }

__device__ __forceinline__ double warp_max_d(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmax(v, __shfl_xor_sync(kFull, v, o));
    return v;
}

// Lane g holds group g's total; returns the bit mask of the `top` best groups (ties: lowest index).  *border: the last
// total kept; *gap: its distance from the first one dropped.
template <typename T>
__device__ uint32_t best_groups(T total, int groups, int top, int lane, T *gap, T *border) {
    int rank = 0;
    T last = -INFINITY, next = -INFINITY;
#pragma unroll 4
    for (int g = 0; g < groups; g++) {
        const T o = __shfl_sync(kFull, total, g);
        rank += (o > total || (o == total && g < lane)) ? 1 : 0;
    }
    const uint32_t keep = __ballot_sync(kFull, lane < groups && rank < top);
    const uint32_t at_last = __ballot_sync(kFull, lane < groups && rank == top - 1), at_next = __ballot_sync(kFull, lane < groups && rank == top);
    if (at_last) last = __shfl_sync(kFull, total, __ffs(at_last) - 1);
    if (at_next) next = __shfl_sync(kFull, total, __ffs(at_next) - 1);
    *border = last;
    *gap = next == -INFINITY ? (T)INFINITY : last - next;
    return keep;
}

// Keys of a lane, largest first: Batcher's odd-even merge sort.
template <int N>
__device__ __forceinline__ void sort_down(uint32_t (&k)[N]) {
#pragma unroll
    for (int p = 1; p < N; p *= 2)
#pragma unroll
        for (int q = p; q >= 1; q /= 2)
#pragma unroll
            for (int j = q % p; j + q < N; j += 2 * q)
#pragma unroll
                for (int i = 0; i < q; i++)
                    if (i + j + q < N && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
                        const uint32_t a = k[i + j], b = k[i + j + q];
                        k[i + j] = max(a, b);
                        k[i + j + q] = min(a, b);
                    }
}

// Order-preserving map of doubles that are not NaN; 0 stands below every value.  The largest of the warp by its two halves: two
// dependent redux, where a butterfly of doubles takes five rounds.
__device__ __forceinline__ unsigned long long key_of(double d) {
    const long long b = __double_as_longlong(d);
    return (unsigned long long)(b ^ (b >> 63 | (long long)0x8000000000000000ull));
}
__device__ __forceinline__ double value_of(unsigned long long k) {
    return __longlong_as_double((long long)(k & 0x8000000000000000ull ? k ^ 0x8000000000000000ull : ~k));
}
__device__ __forceinline__ unsigned long long warp_max_key(unsigned long long k) {
    const uint32_t hi = __reduce_max_sync(kFull, (uint32_t)(k >> 32));
    const uint32_t lo = __reduce_max_sync(kFull, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
    return (unsigned long long)hi << 32 | lo;
}

// Longer rows keep their doubles in local memory: in registers they would cost every warp its share (512 experts, 8192 tokens
// 14.5 us, with 158 registers 17.6).
template <int VPL>
constexpr int kDoubleUnroll = VPL <= 8 ? VPL : 1;

// A row's choices in 64 bits (-inf: not available).
template <int VPL>
__device__ __forceinline__ void choices_in_double(const RouteParams &p, const float *row, int lane, double (&c)[VPL]) {
    double m = -INFINITY, sum = 0.0;
#pragma unroll(kDoubleUnroll<VPL>)
    for (int j = 0; j < VPL; j++) {
        const int e = j * 32 + lane;
        const float x = e < p.experts ? row[e] : -INFINITY;
        const float b = p.bias != nullptr && e < p.experts ? p.bias[e] : 0.f;
        c[j] = (x > -INFINITY && b > -INFINITY) ? (double)x : -INFINITY;
        m = fmax(m, c[j]);
    }
    m = warp_max_d(m);
#pragma unroll(kDoubleUnroll<VPL>)
    for (int j = 0; j < VPL; j++) {
        if (c[j] == -INFINITY) continue;
        c[j] = p.score == FM_SCORE_SOFTMAX ? (c[j] == m ? 1.0 : exp(c[j] - m)) : 1.0 / (1.0 + exp(-c[j]));
        sum += c[j];
    }
    if (p.score == FM_SCORE_SOFTMAX)
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
#pragma unroll(kDoubleUnroll<VPL>)
    for (int j = 0; j < VPL; j++) {
        if (c[j] == -INFINITY) continue;
        if (p.score == FM_SCORE_SOFTMAX) c[j] /= sum;
        if (p.bias != nullptr) c[j] += (double)p.bias[j * 32 + lane];
    }
}

// The groups that survive, where the 32-bit totals do not tell.  A few warps of thousands come here, and a launch waits for them:
// 8192 tokens of 256 experts in 8 groups take 14.6 us without and 15.1 with them (20 when they took the whole row this way).
template <int VPL>
__device__ __noinline__ uint32_t groups_in_double(const RouteParams &p, const float *row, int lane) {
    double c[VPL];
    choices_in_double<VPL>(p, row, lane, c);
    const int size = p.experts / p.groups;
    unsigned long long g1 = 0, g2 = 0;
    for (int g = 0; g < p.groups; g++) {
        unsigned long long m1 = 0, m2 = 0;
#pragma unroll(kDoubleUnroll<VPL>)
        for (int j = 0; j < VPL; j++) {
            if (j * 32 + 31 < g * size || j * 32 >= (g + 1) * size) continue;  // uniform
            const int e = j * 32 + lane;
            const unsigned long long k = e >= g * size && e < (g + 1) * size && c[j] > -INFINITY ? key_of(c[j]) : 0ull;
            m2 = max(m2, min(m1, k));
            m1 = max(m1, k);
        }
        const unsigned long long a = warp_max_key(m1);
        const int holder = __ffs(__ballot_sync(kFull, m1 == a)) - 1;
        const unsigned long long b = p.group_best == 2 ? warp_max_key(lane == holder ? m2 : m1) : 0ull;
        if (lane == g) { g1 = a; g2 = b; }
    }
    const double mine = g1 == 0 ? -INFINITY : g2 == 0 ? value_of(g1) : value_of(g1) + value_of(g2);
    double gap, border;
    return best_groups<double>(mine, p.groups, p.top_groups, lane, &gap, &border);
}

// The whole choice in 64 bits, taken where 32 cannot tell neighbours apart.  Returns the lane's slot's expert (-1: none).
template <int VPL>
__device__ __noinline__ int select_in_double(const RouteParams &p, const float *row, int lane, uint32_t keep) {
    double c[VPL];
    if (p.score == FM_SCORE_SOFTMAX && p.bias == nullptr) {  // the logits decide, as in the kernel: scores underflow, or round to one value
#pragma unroll(kDoubleUnroll<VPL>)
        for (int j = 0; j < VPL; j++) {
            const float x = j * 32 + lane < p.experts ? row[j * 32 + lane] : -INFINITY;
            c[j] = x > -INFINITY ? (double)x : -INFINITY;
        }
    } else {
        choices_in_double<VPL>(p, row, lane, c);
    }
    if (p.groups > 1) {
        const int size = p.experts / p.groups;
        for (int j = 0; j < VPL; j++)
            if (j * 32 + lane < p.experts && !((keep >> ((j * 32 + lane) / size)) & 1)) c[j] = -INFINITY;
    }
    int id = -1;
    for (int s = 0; s < p.top_k; s++) {
        double best = -INFINITY;
        for (int j = 0; j < VPL; j++) best = fmax(best, c[j]);
        best = warp_max_d(best);
        if (best == -INFINITY) break;
        int at = 0x7fffffff;
        for (int j = VPL - 1; j >= 0; j--)
            if (c[j] == best) at = j * 32 + lane;
        at = __reduce_min_sync(kFull, at);
        for (int j = 0; j < VPL; j++)
            if (j * 32 + lane == at) c[j] = -INFINITY;
        if (lane == s) id = at;
    }
    return id;
}

template <int VPL>
__global__ void __launch_bounds__(32 * kRtWarps)
moe_route_kernel(const __grid_constant__ RouteParams p) {
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    const int lane = threadIdx.x & 31, t = blockIdx.x * kRtWarps + (threadIdx.x >> 5);
    if (t >= p.n) return;
    const float *row = p.logits + (size_t)t * (p.experts + p.shared);
    const bool softmax = p.score == FM_SCORE_SOFTMAX;
    const bool by_logit = softmax && p.bias == nullptr;  // order of the logits = order of the scores, without rounding

    // logits; -inf where the expert cannot be chosen (its logit or bias is NaN or -inf)
    float x[VPL];
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < VPL; j++) {
        const int e = j * 32 + lane;
        x[j] = e < p.experts ? __ldg(row + e) : -INFINITY;
    }
#pragma unroll
    for (int j = 0; j < VPL; j++) {
        const int e = j * 32 + lane;
        if (!(x[j] > -INFINITY)) x[j] = -INFINITY;
        if (p.bias != nullptr && e < p.experts && !(__ldg(p.bias + e) > -INFINITY)) x[j] = -INFINITY;
        m = fmaxf(m, x[j]);
    }
    float inv = 0.f, top_score = 1.f;
    uint32_t key[VPL];  // order-preserving; 0: not available
    if (softmax) {
        // the denominator; +inf logits share the weight equally
        m = warp_max(m);
        float sum = 0.f;
        const bool scores = !by_logit || p.groups > 1 || !p.renormalize;  // (renormalised weights need no denominator)
        if (scores) {
#pragma unroll
            for (int j = 0; j < VPL; j++) sum += x[j] > -INFINITY ? (x[j] == m ? 1.f : expf(x[j] - m)) : 0.f;
            sum = warp_sum(sum);
            inv = sum > 0.f ? 1.f / sum : 0.f;
        }
        top_score = inv;
    }
    // error bound of an approximate choice: the score's (softmax: the exponent's rounding grows with its size; sigmoid: the two
    // special functions, 2^-22 each) and the sum's
    const float tol_score = (softmax ? 8e-6f : 1e-6f) * top_score;
    if (by_logit) {
#pragma unroll
        for (int j = 0; j < VPL; j++) key[j] = x[j] > -INFINITY ? key_of(x[j]) : 0u;
    } else {
#pragma unroll
        for (int j = 0; j < VPL; j++) {
            const float s = softmax ? (x[j] == m ? 1.f : expf(x[j] - m)) * inv : fast_sigmoid(x[j]);
            key[j] = x[j] > -INFINITY ? key_of(p.bias != nullptr ? s + __ldg(p.bias + min(j * 32 + lane, p.experts - 1)) : s) : 0u;
        }
    }
    uint32_t keep = 0;  // groups

    if (p.groups > 1) {
        const int size = p.experts / p.groups;
        // lane g gets the best two of group g, from each lane's best two of it; free of branches, so that the groups' chains overlap
        uint32_t g1 = 0, g2 = 0;
        auto best_two = [&](int g, uint32_t m1, uint32_t m2) {
            const uint32_t a = __reduce_max_sync(kFull, m1);
            const int holder = __ffs(__ballot_sync(kFull, m1 == a)) - 1;
            const uint32_t b = __reduce_max_sync(kFull, lane == holder ? m2 : m1);
            g1 = lane == g ? a : g1;
            g2 = lane == g ? b : g2;
        };
        if (size == 32) {  // a register per group
#pragma unroll
            for (int j = 0; j < VPL; j++) best_two(j, key[j], 0u);
        } else if (size % 32 == 0) {  // whole registers per group
            const int regs = size / 32;
            uint32_t m1 = 0, m2 = 0;
            int left = regs, g = 0;
#pragma unroll
            for (int j = 0; j < VPL; j++) {
                m2 = max(m2, min(m1, key[j]));
                m1 = max(m1, key[j]);
                if (--left == 0) {
                    best_two(g++, m1, m2);
                    m1 = m2 = 0; left = regs;
                }
            }
        } else {
            for (int g = 0; g < p.groups; g++) {
                uint32_t m1 = 0, m2 = 0;
#pragma unroll
                for (int j = 0; j < VPL; j++) {
                    if (j * 32 + 31 < g * size || j * 32 >= (g + 1) * size) continue;  // uniform: no expert of the group in register j
                    const int e = j * 32 + lane;
                    const uint32_t k = e >= g * size && e < (g + 1) * size ? key[j] : 0u;
                    m2 = max(m2, min(m1, k));
                    m1 = max(m1, k);
                }
                best_two(g, m1, m2);
            }
        }
        // lane g: the total of group g.  by_logit: the group's best scores are those of its best logits; of one best, compare the
        // logits themselves
        float mine = -INFINITY, size_of = 0.f;  // (size_of: what the total's roundings are relative to)
        if (lane < p.groups && g1 != 0u) {
            auto score = [&](uint32_t k) {
                const float v = value_of(k);
                return by_logit && p.group_best == 2 ? (v == m ? 1.f : expf(v - m)) * inv : v;
            };
            mine = score(g1);
            size_of = fabsf(mine);
            if (p.group_best == 2 && g2 != 0u) {
                const float second = score(g2);
                mine += second;
                size_of += fabsf(second);
            }
        }
        float gap, border;
        keep = best_groups<float>(mine, p.groups, p.top_groups, lane, &gap, &border);
        // Two choices of a group may cancel, so their roundings are taken from their sizes, the largest of any group.  Scores alone
        // (by_logit) do not cancel; below fp32's normal numbers their rounding is absolute.
        const float largest = __uint_as_float(__reduce_max_sync(kFull, __float_as_uint(size_of)));
        if (!(by_logit && p.group_best == 1) && !(gap > (by_logit ? 1.6e-5f * border + 1.2e-38f : 4.f * tol_score + 4.8e-7f * largest)))
            keep = groups_in_double<VPL>(p, row, lane);
        const uint32_t per = ((1u << 20) + size - 1) / size;  // e / size = e * per >> 20 for e < 1024
#pragma unroll
        for (int j = 0; j < VPL; j++)
            if (!((keep >> ((uint32_t)(j * 32 + lane) * per >> 20)) & 1)) key[j] = 0u;
    }

    // Candidates: lane s gets the s-th largest key, its low bits replaced by the index (one redux finds value and holder).  The
    // top_k of them, and as many more as the lost bits and the choice's error leave possible.
    constexpr uint32_t kIndex = 32 * VPL - 1;
#pragma unroll
    for (int j = 0; j < VPL; j++)
        if (key[j] != 0u) key[j] = (key[j] & ~kIndex) | (kIndex - (uint32_t)(j * 32 + lane));
    if constexpr (VPL <= 8) sort_down(key);
    auto take = [&]() {  // the largest key of all, which leaves its lane
        uint32_t best = key[0];
        if constexpr (VPL > 8)
#pragma unroll
            for (int j = 1; j < VPL; j++) best = max(best, key[j]);
        best = __reduce_max_sync(kFull, best);
        if constexpr (VPL <= 8) {
            const bool won = key[0] == best;
#pragma unroll
            for (int j = 0; j + 1 < VPL; j++) key[j] = won ? key[j + 1] : key[j];
            key[VPL - 1] = won ? 0u : key[VPL - 1];
        } else {
#pragma unroll
            for (int j = 0; j < VPL; j++) key[j] = key[j] == best ? 0u : key[j];
        }
        return best;
    };
    // whether a candidate's choice is below another's, whatever the lost bits and the choices' errors are
    auto below = [&](uint32_t a, uint32_t b) {
        return value_of(a | kIndex) + (by_logit ? 0.f : 2.f * tol_score + 2.4e-7f * fabsf(value_of(a))) < value_of(b & ~kIndex);
    };
    uint32_t mine = 0, last = 0, best = 0;
    int nc = 0;
    for (; nc < p.top_k; nc++) {
        best = take();
        if (best == 0u) break;
        if (lane == nc) mine = best;
        last = best;
    }
    bool unsure = false;
    while (best != 0u) {
        best = take();
        if (best == 0u || below(best, last)) break;
        if (nc == 32) { unsure = true; break; }
        if (lane == nc) mine = best;
        nc++;
    }
    // Their exact order, where two neighbours leave a doubt: logits as they are, choices in 64 bits (softmax with a bias: in 32,
    // where that decides).
    int id = lane < nc ? (int)(kIndex - (mine & kIndex)) : -1, rank = lane;
    const uint32_t before = __shfl_up_sync(kFull, mine, 1);
    if (__any_sync(kFull, lane > 0 && lane < nc && !below(mine, before))) {
        const float v0 = id >= 0 ? __ldg(row + id) : -INFINITY;
        rank = 0;
        if (by_logit) {
            for (int j = 0; j < nc; j++) {
                const float o = __shfl_sync(kFull, v0, j);
                const int oe = __shfl_sync(kFull, id, j);
                rank += (o > v0 || (o == v0 && oe < id)) ? 1 : 0;
            }
        } else if (!softmax) {
            double c = -INFINITY;
            if (id >= 0) c = 1.0 / (1.0 + exp(-(double)v0)) + (p.bias != nullptr ? (double)__ldg(p.bias + id) : 0.0);
            for (int j = 0; j < nc; j++) {
                const double o = __shfl_sync(kFull, c, j);
                const int oe = __shfl_sync(kFull, id, j);
                rank += (o > c || (o == c && oe < id)) ? 1 : 0;
            }
        } else {
            const float c = id >= 0 ? (v0 == m ? 1.f : expf(v0 - m)) * inv + __ldg(p.bias + id) : -INFINITY;
            bool near = false;
            for (int j = 0; j < nc; j++) {
                const float o = __shfl_sync(kFull, c, j);
                const int oe = __shfl_sync(kFull, id, j);
                rank += (o > c || (o == c && oe < id)) ? 1 : 0;
                near |= oe != id && !(fabsf(o - c) > 2.f * tol_score + 2.4e-7f * fabsf(c));
            }
            unsure |= __any_sync(kFull, near && id >= 0);
        }
    }
    if (unsure) {
        id = select_in_double<VPL>(p, row, lane, keep);
        rank = lane;
    }
    const bool chosen = id >= 0 && rank < p.top_k;
    const int found = __popc(__ballot_sync(kFull, chosen)), slots = p.top_k + p.shared;

    const float v = chosen ? __ldg(row + id) : -INFINITY;
    float w = 0.f;
    if (!p.renormalize) {
        if (chosen) w = softmax ? (v == m ? 1.f : expf(v - m)) * inv : 1.f / (1.f + expf(-v));
    } else {
        // a common factor drops out: the scores relative to the largest selected one, so that small ones do not underflow
        const float vm = warp_max(v);
        if (chosen) {
            const float rel = v == vm ? 1.f : expf(v - vm);
            w = softmax ? rel : vm > 0.f ? 1.f / (1.f + expf(-v)) : rel / (1.f + expf(v));
        }
        const float tot = warp_sum(w);
        w = tot > 0.f ? w / tot : 0.f;
    }
    int *ids = p.ids + (size_t)t * slots;
    float *weights = p.weights + (size_t)t * slots;
    if (chosen) { ids[rank] = id; weights[rank] = w * p.scale; }
    if (lane >= found && lane < p.top_k) { ids[lane] = -1; weights[lane] = 0.f; }
    if (p.shared && lane == 0) {
        ids[p.top_k] = p.experts;
        weights[p.top_k] = 1.f / (1.f + expf(-__ldg(row + p.experts)));
    }
}

}  // namespace

int launch_moe_route(const RouteParams &p, cudaStream_t st) {
    const dim3 grid((p.n + kRtWarps - 1) / kRtWarps), block(32 * kRtWarps);
    cudaError_t e;
    if (p.experts <= 32) e = launch_dependent(moe_route_kernel<1>, grid, block, 0, st, p);
    else if (p.experts <= 64) e = launch_dependent(moe_route_kernel<2>, grid, block, 0, st, p);
    else if (p.experts <= 128) e = launch_dependent(moe_route_kernel<4>, grid, block, 0, st, p);
    else if (p.experts <= 256) e = launch_dependent(moe_route_kernel<8>, grid, block, 0, st, p);
    else if (p.experts <= 512) e = launch_dependent(moe_route_kernel<16>, grid, block, 0, st, p);
    else e = launch_dependent(moe_route_kernel<32>, grid, block, 0, st, p);
    return e == cudaSuccess ? 1 : -1;
}

}  // namespace fm
