// route.cu -- the router of the routed linears and the weighted sum behind
// them: top-k experts per token with their softmax weights, the plan (rows
// sorted by expert, stably), and out = residual + sum_j weight_j y[slot_j].
//
// Router.  choice j of token t is its j-th largest finite logit, ties to the
// lower index; the weight is exp(l - max) over the sum of the chosen ones or of
// all finite ones.  The plan is a stable counting sort of the (token, choice)
// items by expert: item i of expert e goes to
//   offsets[e] + (items of e in earlier blocks) + (items of e before i in its block).
// route_topk_kernel writes each item's rank in its block (into `slots`) and the
// block's histogram; route_plan_kernel turns the histograms into positions.  It
// needs no third launch for the scan: each block sums the histogram columns it
// needs itself (experts x blocks integers out of L2).  One block's worth of
// tokens is planned by the first kernel alone, in one launch.
#include <algorithm>

#include "samq_internal.hpp"

namespace samq {
namespace {

constexpr int kRouteThreads = 256;
constexpr int kRouteWarps = kRouteThreads / 32;
constexpr int kMaxExperts = 1024;
constexpr float kNegInf = -__builtin_huge_valf();

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Exclusive prefix sum of counts[0 .. n) in shared memory by one warp, n a
// multiple of nothing: counts[i] becomes the sum before i; returns the total.
__device__ __forceinline__ int warp_exclusive_scan(int* counts, int n, int lane) {
    int carry = 0;
    for (int base = 0; base < n; base += 32) {
        const int v = base + lane < n ? counts[base + lane] : 0;
        int s = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += u;
        }
        if (base + lane < n) counts[base + lane] = carry + s - v;
        carry += __shfl_sync(0xffffffffu, s, 31);
    }
    return carry;
}

// One warp per token: V = ceil(experts / 32) logits per lane in registers
// (expert 32 v + lane), top_k rounds of a warp-wide maximum.
template <int V>
__device__ __forceinline__ void route_token(const float* __restrict__ row, int experts, int top_k, bool normalize,
                                            float* __restrict__ weights, int* __restrict__ ids, int* picked,
                                            int lane) {
    float v[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int e = 32 * i + lane;
        const float l = e < experts ? __ldg(row + e) : kNegInf;
        v[i] = fabsf(l) < __builtin_huge_valf() ? l : kNegInf;  // NaN and infinities are not eligible
    }
    float best = kNegInf;
#pragma unroll
    for (int i = 0; i < V; ++i) best = fmaxf(best, v[i]);
    best = warp_max(best);
    float sum = 0.0f;
    if (!normalize && best > kNegInf) {
#pragma unroll
        for (int i = 0; i < V; ++i) sum += expf(v[i] - best);
        sum = warp_sum(sum);
    }
    // The lane with choice j keeps its logit and expert (top_k <= 32).
    float mine = kNegInf;
    int mine_id = -1;
    for (int j = 0; j < top_k; ++j) {
        float m = kNegInf;
        int e = kMaxExperts;
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (v[i] > m) {  // ascending expert order: the first of equals stays
                m = v[i];
                e = 32 * i + lane;
            }
        const float top = warp_max(m);
        if (top == kNegInf) break;
        const int id = __reduce_min_sync(0xffffffffu, m == top ? e : kMaxExperts);
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (32 * i + lane == id) v[i] = kNegInf;
        if (lane == j) {
            mine = top;
            mine_id = id;
        }
    }
    const float p = mine_id >= 0 ? expf(mine - best) : 0.0f;
    if (normalize) sum = warp_sum(p);
    if (lane < top_k) {
        weights[lane] = mine_id >= 0 ? p / sum : 0.0f;
        ids[lane] = mine_id;
        picked[lane] = mine_id;
    }
}

// Block b routes tokens [b * per_block, ...).  SINGLE: the only block, which
// also writes the plan.  Dynamic shared memory: picked[per_block * top_k],
// counts[experts].
template <int V, bool SINGLE>
__global__ void __launch_bounds__(kRouteThreads) route_topk_kernel(const float* __restrict__ logits, int tokens,
                                                                   int experts, int64_t ld, int top_k, int normalize,
                                                                   int per_block, float* __restrict__ weights,
                                                                   int* __restrict__ ids, int* __restrict__ offsets,
                                                                   int* __restrict__ rows, int* __restrict__ slots,
                                                                   int* __restrict__ hist) {
    extern __shared__ int route_smem[];
    int* picked = route_smem;
    int* counts = picked + per_block * top_k;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t0 = blockIdx.x * per_block, count = min(per_block, tokens - t0);
    for (int e = threadIdx.x; e < experts; e += kRouteThreads) counts[e] = 0;
    pdl_wait();
    pdl_trigger();
    for (int t = warp; t < count; t += kRouteWarps) {
        const int64_t token = t0 + t;
        route_token<V>(logits + token * ld, experts, top_k, normalize != 0, weights + token * top_k,
                       ids + token * top_k, picked + t * top_k, lane);
    }
    __syncthreads();
    // Ranks in (token, choice) order by one warp, 32 items at a time.
    const int items = count * top_k;
    int* my_slots = slots + static_cast<int64_t>(t0) * top_k;
    if (warp == 0) {
        for (int base = 0; base < items; base += 32) {
            const int e = base + lane < items ? picked[base + lane] : -1;
            const unsigned same = __match_any_sync(0xffffffffu, e);
            const int before = __popc(same & ((1u << lane) - 1u));
            const int rank = (e >= 0 ? counts[e] : 0) + before;
            __syncwarp();
            if (e >= 0 && before == 0) counts[e] = rank + __popc(same);
            __syncwarp();
            if (base + lane < items) {
                if (SINGLE) picked[base + lane] = e >= 0 ? (rank << 10) | e : -1;
                else my_slots[base + lane] = e >= 0 ? rank : -1;
            }
        }
        if (SINGLE) {
            const int total = warp_exclusive_scan(counts, experts, lane);
            if (lane == 0) offsets[experts] = total;
        }
    }
    __syncthreads();
    if (!SINGLE) {
        for (int e = threadIdx.x; e < experts; e += kRouteThreads)
            hist[static_cast<int64_t>(e) * gridDim.x + blockIdx.x] = counts[e];
        return;
    }
    for (int e = threadIdx.x; e < experts; e += kRouteThreads) offsets[e] = counts[e];
    for (int i = threadIdx.x; i < items; i += kRouteThreads) {
        const int p = picked[i];
        if (p >= 0) {
            const int at = counts[p & 1023] + (p >> 10);
            rows[at] = i / top_k;
            slots[i] = at;
        } else {
            slots[i] = -1;
        }
    }
    // Rows behind the plan: as many as there are empty choices.
    __syncthreads();
    if (warp == 0) {
        int kept = 0;
        for (int i = lane; i < items; i += 32) kept += picked[i] >= 0;
        kept = __reduce_add_sync(0xffffffffu, kept);
        for (int i = kept + lane; i < items; i += 32) rows[i] = -1;
    }
}

// Positions from the block histograms.  Dynamic shared memory: start[experts]
// (totals, then offsets), before[experts].
__global__ void __launch_bounds__(kRouteThreads) route_plan_kernel(const int* __restrict__ hist, int tokens,
                                                                   int experts, int top_k, int per_block,
                                                                   const int* __restrict__ ids,
                                                                   int* __restrict__ offsets, int* __restrict__ rows,
                                                                   int* __restrict__ slots) {
    extern __shared__ int route_smem[];
    int* start = route_smem;
    int* before = start + experts;
    __shared__ int s_total;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int blocks = gridDim.x;
    pdl_wait();
    pdl_trigger();
    for (int e = warp; e < experts; e += kRouteWarps) {
        int all = 0, mine = 0;
        for (int b = lane; b < blocks; b += 32) {
            const int c = hist[static_cast<int64_t>(e) * blocks + b];
            all += c;
            mine += b < static_cast<int>(blockIdx.x) ? c : 0;
        }
        all = __reduce_add_sync(0xffffffffu, all);
        mine = __reduce_add_sync(0xffffffffu, mine);
        if (lane == 0) {
            start[e] = all;
            before[e] = mine;
        }
    }
    __syncthreads();
    if (warp == 0) {
        const int total = warp_exclusive_scan(start, experts, lane);
        if (lane == 0) s_total = total;
    }
    __syncthreads();
    if (blockIdx.x == 0) {
        for (int e = threadIdx.x; e < experts; e += kRouteThreads) offsets[e] = start[e];
        if (threadIdx.x == 0) offsets[experts] = s_total;
    }
    const int t0 = blockIdx.x * per_block, count = min(per_block, tokens - t0);
    const int64_t base = static_cast<int64_t>(t0) * top_k;
    for (int i = threadIdx.x; i < count * top_k; i += kRouteThreads) {
        const int e = ids[base + i];
        if (e >= 0) {
            const int at = start[e] + before[e] + slots[base + i];
            rows[at] = t0 + i / top_k;
            slots[base + i] = at;
        }
        if (base + i >= s_total) rows[base + i] = -1;  // no plan row lies there
    }
}

// Tokens of one block: few enough that a prefill fills the GPU, many enough
// that the histograms stay small, and at most kMaxItems choices.
constexpr int kMaxItems = 49152;  // 4 bytes each of shared memory beside the histogram
int route_tokens_per_block(int64_t tokens, int top_k) {
    if (tokens <= 64) return 64;
    return static_cast<int>(std::min<int64_t>(std::max<int64_t>((tokens + 255) / 256, 16), kMaxItems / top_k));
}

template <int V>
void run_route(const float* logits, int tokens, int experts, int64_t ld, int top_k, int normalize, int per_block,
               int blocks, float* weights, int* ids, int* offsets, int* rows, int* slots, int* hist,
               DeviceState& state, cudaStream_t stream) {
    const size_t smem = (static_cast<size_t>(per_block) * top_k + experts) * sizeof(int);
    auto kernel = blocks == 1 ? route_topk_kernel<V, true> : route_topk_kernel<V, false>;
    set_smem_limit_once(state, reinterpret_cast<const void*>(kernel), 200 * 1024, "cudaFuncSetAttribute(route smem)");
    launch_pdl(kernel, dim3(blocks), dim3(kRouteThreads), smem, stream, "route_topk_kernel launch", logits, tokens,
               experts, ld, top_k, normalize, per_block, weights, ids, offsets, rows, slots, hist);
}

// 8 columns of a row of Y as floats.
__device__ __forceinline__ void load_y(const __half* p, float (&v)[8]) {
    const uint4 raw = __ldg(reinterpret_cast<const uint4*>(p));
    const __half2* h = reinterpret_cast<const __half2*>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(h[i]);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void load_y(const float* p, float (&v)[4]) {
    const float4 f = __ldg(reinterpret_cast<const float4*>(p));
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
}

// One 16-byte column group of one token per thread.
template <class T>
__global__ void __launch_bounds__(256) combine_kernel(const T* __restrict__ y, int64_t y_rows, int64_t ldy,
                                                      const int* __restrict__ slots, const float* __restrict__ weights,
                                                      int64_t tokens, int top_k, int64_t width, const float* residual,
                                                      int64_t ldr, float* out, int64_t ldo) {
    constexpr int C = 16 / sizeof(T);
    pdl_wait();
    pdl_trigger();
    const int64_t per_row = width / C;
    const int64_t units = tokens * per_row;
    for (int64_t u = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; u < units;
         u += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        const int64_t t = u / per_row, c = (u - t * per_row) * C;
        float acc[C] = {};
        for (int j = 0; j < top_k; ++j) {
            const int slot = __ldg(slots + t * top_k + j);
            if (slot < 0 || slot >= y_rows) continue;
            const float w = __ldg(weights + t * top_k + j);
            float v[C];
            load_y(y + static_cast<int64_t>(slot) * ldy + c, v);
#pragma unroll
            for (int i = 0; i < C; ++i) acc[i] = fmaf(w, v[i], acc[i]);
        }
#pragma unroll
        for (int i = 0; i < C; i += 4) {
            float4 r = residual ? *reinterpret_cast<const float4*>(residual + t * ldr + c + i)
                                : make_float4(0.f, 0.f, 0.f, 0.f);
            r.x += acc[i];
            r.y += acc[i + 1];
            r.z += acc[i + 2];
            r.w += acc[i + 3];
            *reinterpret_cast<float4*>(out + t * ldo + c + i) = r;
        }
    }
}

}  // namespace

size_t route_workspace_bytes(int64_t tokens, int experts, int top_k) {
    const int per_block = route_tokens_per_block(tokens, top_k);
    const int64_t blocks = (tokens + per_block - 1) / per_block;
    return blocks > 1 ? static_cast<size_t>(blocks) * experts * sizeof(int) : 0;
}

void launch_route(const float* logits, int64_t tokens, int experts, int64_t ld, int top_k, int normalize,
                  float* weights, int32_t* ids, int32_t* offsets, int32_t* rows, int32_t* slots, void* workspace,
                  DeviceState& state, cudaStream_t stream) {
    const int per_block = route_tokens_per_block(tokens, top_k);
    const int blocks = static_cast<int>(std::max<int64_t>((tokens + per_block - 1) / per_block, 1));
    int* hist = static_cast<int*>(workspace);
    auto run = [&](auto width) {
        constexpr int V = decltype(width)::value;
        run_route<V>(logits, static_cast<int>(tokens), experts, ld, top_k, normalize, per_block, blocks, weights, ids,
                     offsets, rows, slots, hist, state, stream);
    };
    if (experts <= 64) run(std::integral_constant<int, 2>());
    else if (experts <= 128) run(std::integral_constant<int, 4>());
    else if (experts <= 256) run(std::integral_constant<int, 8>());
    else run(std::integral_constant<int, 32>());
    if (blocks > 1)
        launch_pdl(route_plan_kernel, dim3(blocks), dim3(kRouteThreads), 2 * experts * sizeof(int), stream,
                   "route_plan_kernel launch", static_cast<const int*>(hist), static_cast<int>(tokens), experts, top_k,
                   per_block, static_cast<const int*>(ids), offsets, rows, slots);
}

void launch_combine(const void* y, int y_type, int64_t y_rows, int64_t ldy, const int32_t* slots, const float* weights,
                    int64_t tokens, int top_k, int64_t width, const float* residual, int64_t ldr, float* out,
                    int64_t ldo, DeviceState& state, cudaStream_t stream) {
    const int64_t units = tokens * (width / (y_type == SAMQ_TYPE_F16 ? 8 : 4));
    const unsigned grid =
        static_cast<unsigned>(std::min<int64_t>((units + 255) / 256, static_cast<int64_t>(state.sm_count) * 64));
    if (y_type == SAMQ_TYPE_F16)
        launch_pdl(combine_kernel<__half>, dim3(grid), dim3(256), 0, stream, "combine_kernel launch",
                   static_cast<const __half*>(y), y_rows, ldy, slots, weights, tokens, top_k, width, residual, ldr,
                   out, ldo);
    else
        launch_pdl(combine_kernel<float>, dim3(grid), dim3(256), 0, stream, "combine_kernel launch",
                   static_cast<const float*>(y), y_rows, ldy, slots, weights, tokens, top_k, width, residual, ldr,
                   out, ldo);
}

}  // namespace samq
