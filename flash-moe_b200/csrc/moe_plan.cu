// Around the experts' products: which pairs (token, slot) go to which expert, and the weighted sum behind them.
#include <math.h>

#include <algorithm>

#include "fm_device.cuh"
#include "fm_internal.h"

namespace fm {

namespace {

constexpr int kPlanThreads = 1024;  // one thread per expert in the scan: at most 1024 experts held

// inclusive sums of two counts over the block
__device__ __forceinline__ void block_scan2(int &a, int &b, int *s_a, int *s_b) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
        if (lane >= o) { a += x; b += y; }
    }
    if (lane == 31) { s_a[warp] = a; s_b[warp] = b; }
    __syncthreads();
    if (warp == 0) {
        int x = s_a[lane], y = s_b[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, x, o), v = __shfl_up_sync(0xffffffffu, y, o);
            if (lane >= o) { x += u; y += v; }
        }
        s_a[lane] = x; s_b[lane] = y;
    }
    __syncthreads();
    if (warp > 0) { a += s_a[warp - 1]; b += s_b[warp - 1]; }
}

// A counting sort of the pairs by expert, in one CTA.  Within an expert the order is that of the atomics and changes from
// run to run; nothing depends on it, since a pair's products do not depend on its neighbours.
__global__ void __launch_bounds__(kPlanThreads)
moe_plan_kernel(const int *__restrict__ ids, int pairs, int first_expert, int num_experts, int tile, MoePlan plan) {
    __shared__ int s_count[kPlanThreads], s_a[32], s_b[32];
    const int tid = threadIdx.x;
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    s_count[tid] = 0;
    __syncthreads();
    // eight ids per thread in flight
    auto each = [&](auto &&use) {
        for (int p0 = tid; p0 < pairs; p0 += 8 * kPlanThreads) {
            int e[8];
#pragma unroll
            for (int i = 0; i < 8; i++) e[i] = p0 + i * kPlanThreads < pairs ? local_expert(__ldg(ids + p0 + i * kPlanThreads), first_expert, num_experts) : -1;
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (e[i] >= 0) use(e[i], p0 + i * kPlanThreads);
        }
    };
    each([&](int e, int) { atomicAdd(s_count + e, 1); });
    __syncthreads();
    const int count = s_count[tid], tiles = (count + tile - 1) / tile;
    int end = count, tend = tiles;
    block_scan2(end, tend, s_a, s_b);
    const int start = end - count, tstart = tend - tiles;
    s_count[tid] = start;  // from here on the next free position
    // jobs of equal size (in the tensor cores' steps of 16 where they are that large), not full ones and a remainder
    int size = tiles > 0 ? (count + tiles - 1) / tiles : 0;
    if (tile > 16) size = (size + 15) / 16 * 16;
    for (int i = 0; i < tiles; i++) plan.jobs[tstart + i] = make_int4(tid, start + i * size, min(size, count - i * size), 0);  // (size <= tile: none is empty)
    if (tid == kPlanThreads - 1) { plan.njobs[0] = tend; plan.njobs[1] = end; }
    __syncthreads();
    each([&](int e, int p) { plan.pair_of[atomicAdd(s_count + e, 1)] = p; });
}

// One CTA per token.  The slots are summed in their order, so the result does not depend on the launch; eight of their loads
// are in flight at a time.  Up to two tokens per SM get four columns per thread (the row at once), more get small CTAs, four
// to an SM, which cover each other's meeting points.  Measured, large then small CTAs, whole calls with 8 slots of 4096 columns
// and experts of 64 inputs: 148 tokens 92 and 97 us, 296 tokens 117 and 118, 400 tokens 133 and 130, 1000 tokens 234 and 222;
// 4096 tokens with 10 slots, by itself: 180 and 150 us (4.9 TB/s).  A row split over a cluster of CTAs, with the ids fetched
// before the products end, took the same time at one token.
constexpr int kCombineThreads = 1024, kCombineThreadsMany = 256;
constexpr int kCombineBatch = 8;

__global__ void __launch_bounds__(kCombineThreads)
moe_combine_kernel(const float *__restrict__ y, const int *__restrict__ ids, const float *__restrict__ weights, int top_k, int first_expert,
                   int num_experts, int hidden, const float *residual, const uint16_t *__restrict__ norm_w, float eps, float *h_out, float *h_norm) {
    __shared__ float s_w[32], s_sq[32];
    __shared__ int s_slot[32];
    __shared__ int s_n;
    const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nwarps = blockDim.x >> 5, step = blockDim.x * 4;
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    if (warp == 0) {  // the slots that have an expert here
        const bool here = lane < top_k && local_expert(ids[(size_t)t * top_k + lane], first_expert, num_experts) >= 0;
        const unsigned m = __ballot_sync(0xffffffffu, here);
        if (here) {
            const int at = __popc(m & ((1u << lane) - 1));
            s_slot[at] = lane;
            s_w[at] = weights[(size_t)t * top_k + lane];
        }
        if (lane == 0) s_n = __popc(m);
    }
    __syncthreads();
    const int ns = s_n;
    const float *yt = y + (size_t)t * top_k * hidden;
    float sq = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = tid * 4; i < hidden; i += step) {
        const float4 r = residual != nullptr ? *reinterpret_cast<const float4 *>(residual + (size_t)t * hidden + i) : make_float4(0.f, 0.f, 0.f, 0.f);
        a = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int s0 = 0; s0 < ns; s0 += kCombineBatch) {
            float4 v[kCombineBatch];
#pragma unroll
            for (int s = 0; s < kCombineBatch; s++)
                if (s0 + s < ns) v[s] = __ldg(reinterpret_cast<const float4 *>(yt + (size_t)s_slot[s0 + s] * hidden + i));
#pragma unroll
            for (int s = 0; s < kCombineBatch; s++)
                if (s0 + s < ns) {
                    const float w = s_w[s0 + s];
                    a.x = fmaf(w, v[s].x, a.x); a.y = fmaf(w, v[s].y, a.y); a.z = fmaf(w, v[s].z, a.z); a.w = fmaf(w, v[s].w, a.w);
                }
        }
        a.x += r.x; a.y += r.y; a.z += r.z; a.w += r.w;
        *reinterpret_cast<float4 *>(h_out + (size_t)t * hidden + i) = a;
        sq += (a.x * a.x + a.y * a.y) + (a.z * a.z + a.w * a.w);
    }
    if (h_norm == nullptr) return;
    sq = warp_sum(sq);
    if (lane == 0) s_sq[warp] = sq;
    __syncthreads();
    float tot = 0.f;
    for (int w = 0; w < nwarps; w++) tot += s_sq[w];
    const float inv = 1.0f / sqrtf(tot / hidden + eps);
    for (int i = tid * 4; i < hidden; i += step) {
        const float4 h = hidden <= step ? a : *reinterpret_cast<const float4 *>(h_out + (size_t)t * hidden + i);  // its own columns
        uint2 wb = make_uint2(0x3f803f80u, 0x3f803f80u);
        if (norm_w != nullptr) wb = __ldg(reinterpret_cast<const uint2 *>(norm_w + i));
        *reinterpret_cast<float4 *>(h_norm + (size_t)t * hidden + i) =
            make_float4(h.x * inv * __uint_as_float(wb.x << 16), h.y * inv * __uint_as_float(wb.x & 0xffff0000u),
                        h.z * inv * __uint_as_float(wb.y << 16), h.w * inv * __uint_as_float(wb.y & 0xffff0000u));
    }
}

}  // namespace

int launch_moe_plan(const int *ids, int pairs, int first_expert, int num_experts, int tile, const MoePlan &plan, cudaStream_t st) {
    return launch_dependent(moe_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, ids, pairs, first_expert, num_experts, tile, plan) == cudaSuccess ? 1 : -1;
}

int launch_moe_combine(const float *y, const int *ids, const float *weights, int n, int top_k, int first_expert, int num_experts, int hidden,
                       const float *residual, const uint16_t *norm_w, float eps, float *h_out, float *h_norm, int sm_count, cudaStream_t st) {
    return launch_dependent(moe_combine_kernel, dim3(n), dim3(std::min(n > 2 * sm_count ? kCombineThreadsMany : kCombineThreads, (hidden / 4 + 31) / 32 * 32)), 0, st, y, ids,
                            weights, top_k, first_expert, num_experts, hidden, residual, norm_w, eps, h_out, h_norm) == cudaSuccess ? 1 : -1;
}

}  // namespace fm
