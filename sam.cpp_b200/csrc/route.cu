// route.cu -- the router of the routed linears and the weighted sum behind
// them: top-k experts per token with their softmax weights, the plan (rows
// sorted by expert, stably), and out = residual + sum_j weight_j y[slot_j].
//
// Router.  choice j of token t is its j-th largest finite logit, ties to the
// lower index; the weight is exp(l - max) over the sum of the chosen ones or of
// all finite ones.  A warp per token keeps the logits as order-preserving integers
// in registers, so a round is two warp reductions of one instruction each.
// The plan is a stable counting sort of the (token, choice) items by expert: item
// i of expert e goes to
//   offsets[e] + (items of e in earlier blocks) + (items of e before i in its block).
// Up to 64 tokens one block does all of it in one launch, where latency is all
// there is.  More take three: route_topk_kernel leaves each item's rank in its block
// (in `slots`) and the block's histogram, route_scan_kernel turns each expert's
// histogram row into prefix sums (a warp per expert), route_place_kernel adds up.
// 16384 tokens, 128 experts, top 8 take 18.8 us, most of them in the first, where
// latency and not a unit's rate is the bound: 43% of the issue slots, 6% of the HBM;
// the warps wait for the reductions and for one warp's ranking.
#include <algorithm>

#include "samq_internal.hpp"

namespace samq {
namespace {

constexpr int kTopkThreads = 512;   // of a block of many
constexpr int kPlaceThreads = 256;
constexpr int kMaxExperts = 1024;

// Finite floats as unsigned integers in the same order, above 0; 0: not eligible
// (-0 sorts below +0: they are made equal first).
__device__ __forceinline__ uint32_t order_key(float l) {
    if (!(fabsf(l) < __builtin_huge_valf())) return 0;
    const uint32_t b = __float_as_uint(l + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
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
__device__ __forceinline__ void load_keys(const float* __restrict__ row, int experts, int lane, uint32_t (&key)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int e = 32 * i + lane;
        key[i] = e < experts ? order_key(__ldg(row + e)) : 0;
    }
}

// Up to 8 logits a lane are sorted once (adjacent exchanges on strict order: the
// lower expert of equals stays first), so that a round only looks at the lanes'
// heads and the winner moves up: 18.8 us for 16384 tokens, 128 experts, top 8 against
// 21.5 when every round scans the lane's logits, which more logits do.
template <int V>
__device__ __forceinline__ void route_token(uint32_t (&key)[V], int top_k, bool normalize, float* __restrict__ weights,
                                            int* __restrict__ ids, int* picked, int lane) {
    constexpr bool kSorted = V <= 8;
    int id[V];
#pragma unroll
    for (int i = 0; i < V; ++i) id[i] = 32 * i + lane;
    if constexpr (kSorted) {
#pragma unroll
        for (int n = V - 1; n > 0; --n)
#pragma unroll
            for (int i = 0; i < n; ++i) {
                const bool swap = key[i + 1] > key[i];
                const uint32_t high = max(key[i], key[i + 1]), low = min(key[i], key[i + 1]);
                const int first = swap ? id[i + 1] : id[i], second = swap ? id[i] : id[i + 1];
                key[i] = high;
                key[i + 1] = low;
                id[i] = first;
                id[i + 1] = second;
            }
    }
    auto head = [&](int& e) {
        if constexpr (kSorted) {
            e = id[0];
            return key[0];
        } else {
            uint32_t m = 0;
            e = kMaxExperts;
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (key[i] > m) {  // ascending expert order: the first of equals stays
                    m = key[i];
                    e = id[i];
                }
            return m;
        }
    };
    int e;
    uint32_t m = head(e);
    const uint32_t best = __reduce_max_sync(0xffffffffu, m);
    const float top = key_value(best);
    float sum = 0.0f;
    if (!normalize && best) {
#pragma unroll
        for (int i = 0; i < V; ++i) sum += key[i] ? expf(key_value(key[i]) - top) : 0.0f;
        sum = warp_sum(sum);
    }
    // The lane with choice j keeps its logit and expert (top_k <= 32).
    uint32_t mine = 0;
    int mine_id = -1;
    uint32_t largest = best;
    for (int j = 0; largest;) {
        const int winner = __reduce_min_sync(0xffffffffu, m == largest ? e : kMaxExperts);
        if (lane == j) {
            mine = largest;
            mine_id = winner;
        }
        if (++j == top_k) break;
        if constexpr (kSorted) {
            if (e == winner) {
#pragma unroll
                for (int i = 0; i + 1 < V; ++i) {
                    key[i] = key[i + 1];
                    id[i] = id[i + 1];
                }
                key[V - 1] = 0;
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (id[i] == winner) key[i] = 0;
        }
        m = head(e);
        largest = __reduce_max_sync(0xffffffffu, m);
    }
    const float p = mine ? expf(key_value(mine) - top) : 0.0f;
    if (normalize) sum = warp_sum(p);
    if (lane < top_k) {
        weights[lane] = mine ? p / sum : 0.0f;
        ids[lane] = mine_id;
        picked[lane] = mine_id;
    }
}

// Block b routes tokens [b * per_block, ...).  SINGLE: the only block, which
// also writes the plan.  Dynamic shared memory: picked[per_block * top_k],
// counts[experts].
template <int V, bool SINGLE>
__global__ void __launch_bounds__(V > 8 ? 512 : 1024)
route_topk_kernel(const float* __restrict__ logits, int tokens, int experts, int64_t ld, int top_k, int normalize,
                  int per_block, float* __restrict__ weights, int* __restrict__ ids, int* __restrict__ offsets,
                  int* __restrict__ rows, int* __restrict__ slots, int* __restrict__ hist) {
    extern __shared__ int route_smem[];
    int* picked = route_smem;
    int* counts = picked + per_block * top_k;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const int t0 = blockIdx.x * per_block, count = min(per_block, tokens - t0);
    for (int e = threadIdx.x; e < experts; e += blockDim.x) counts[e] = 0;
    pdl_wait();
    pdl_trigger();
    uint32_t key[V], next[V];
    if (warp < count) load_keys<V>(logits + static_cast<int64_t>(t0 + warp) * ld, experts, lane, next);
    for (int t = warp; t < count; t += warps) {
        const int64_t token = t0 + t;
#pragma unroll
        for (int i = 0; i < V; ++i) key[i] = next[i];
        if (t + warps < count) load_keys<V>(logits + (token + warps) * ld, experts, lane, next);
        route_token<V>(key, top_k, normalize != 0, weights + token * top_k, ids + token * top_k, picked + t * top_k, lane);
    }
    __syncthreads();
    // Ranks in (token, choice) order by one warp, 32 items at a time.
    const int items = count * top_k;
    int* my_slots = slots + static_cast<int64_t>(t0) * top_k;
    if (warp == 0) {
        int kept = 0;
        for (int base = 0; base < items; base += 32) {
            const int e = base + lane < items ? picked[base + lane] : -1;
            const unsigned same = __match_any_sync(0xffffffffu, e);
            const int before = __popc(same & ((1u << lane) - 1u));
            const int rank = (e >= 0 ? counts[e] : 0) + before;
            __syncwarp();
            if (e >= 0 && before == 0) counts[e] = rank + __popc(same);
            __syncwarp();
            if (base + lane < items) {
                if constexpr (SINGLE) picked[base + lane] = e >= 0 ? (rank << 10) | e : -1;
                else my_slots[base + lane] = e >= 0 ? rank : -1;
            }
            kept += __popc(__ballot_sync(0xffffffffu, e >= 0));
        }
        if constexpr (SINGLE) {
            const int total = warp_exclusive_scan(counts, experts, lane);
            if (lane == 0) offsets[experts] = total;
            for (int i = kept + lane; i < items; i += 32) rows[i] = -1;  // behind the plan
        }
    }
    __syncthreads();
    if constexpr (!SINGLE) {
        for (int e = threadIdx.x; e < experts; e += blockDim.x)
            hist[static_cast<int64_t>(e) * gridDim.x + blockIdx.x] = counts[e];
    } else {
        for (int e = threadIdx.x; e < experts; e += blockDim.x) offsets[e] = counts[e];
        for (int i = threadIdx.x; i < items; i += blockDim.x) {
            const int p = picked[i];
            if (p >= 0) {
                const int at = counts[p & 1023] + (p >> 10);
                rows[at] = i / top_k;
                slots[i] = at;
            } else {
                slots[i] = -1;
            }
        }
    }
}

// hist[e][0 .. blocks) becomes its exclusive prefix sums, totals[e] the sum; a warp per expert.
__global__ void __launch_bounds__(kPlaceThreads) route_scan_kernel(int* __restrict__ hist, int blocks, int experts,
                                                                   int* __restrict__ totals) {
    const int e = (blockIdx.x * kPlaceThreads + threadIdx.x) >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    pdl_trigger();
    if (e >= experts) return;
    int* row = hist + static_cast<int64_t>(e) * blocks;
    int carry = 0;
    for (int base = 0; base < blocks; base += 128) {
        int v[4], sum = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int b = base + 4 * lane + j;
            v[j] = b < blocks ? row[b] : 0;
            sum += v[j];
        }
        int s = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += u;
        }
        int at = carry + s - sum;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (base + 4 * lane + j < blocks) row[base + 4 * lane + j] = at;
            at += v[j];
        }
        carry += __shfl_sync(0xffffffffu, s, 31);
    }
    if (lane == 0) totals[e] = carry;
}

// Positions of the items of block blockIdx.x * kPlaceThreads ...  Dynamic shared memory: start[experts].
__global__ void __launch_bounds__(kPlaceThreads) route_place_kernel(const int* __restrict__ hist,
                                                                    const int* __restrict__ totals, int64_t items,
                                                                    int experts, int top_k, int per_block, int blocks,
                                                                    const int* __restrict__ ids,
                                                                    int* __restrict__ offsets, int* __restrict__ rows,
                                                                    int* __restrict__ slots) {
    extern __shared__ int route_smem[];
    int* start = route_smem;
    __shared__ int s_total;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    pdl_trigger();
    for (int e = threadIdx.x; e < experts; e += kPlaceThreads) start[e] = __ldg(totals + e);
    __syncthreads();
    if (warp == 0) {
        const int total = warp_exclusive_scan(start, experts, lane);
        if (lane == 0) s_total = total;
    }
    __syncthreads();
    if (blockIdx.x == 0) {
        for (int e = threadIdx.x; e < experts; e += kPlaceThreads) offsets[e] = start[e];
        if (threadIdx.x == 0) offsets[experts] = s_total;
    }
    const int64_t i = static_cast<int64_t>(blockIdx.x) * kPlaceThreads + threadIdx.x;
    if (i >= items) return;
    const int e = ids[i];
    if (e >= 0) {
        const int token = static_cast<int>(i / top_k);
        const int at = start[e] + __ldg(hist + static_cast<int64_t>(e) * blocks + token / per_block) + slots[i];
        rows[at] = token;
        slots[i] = at;
    }
    if (i >= s_total) rows[i] = -1;  // no plan row lies there
}

// Tokens of one block: one block up to 64; beyond, few enough that a prefill
// fills the GPU, at most 512 blocks (the histograms stay small), and at most
// kMaxItems choices.
constexpr int kSingleTokens = 64;
constexpr int kMaxItems = 49152;  // 4 bytes each of shared memory beside the histogram
int route_tokens_per_block(int64_t tokens, int top_k) {
    if (tokens <= kSingleTokens) return kSingleTokens;
    return static_cast<int>(std::min<int64_t>(std::max<int64_t>((tokens + 511) / 512, 16), kMaxItems / top_k));
}

template <int V>
void run_route(const float* logits, int tokens, int experts, int64_t ld, int top_k, int normalize, int per_block,
               int blocks, float* weights, int* ids, int* offsets, int* rows, int* slots, int* hist,
               DeviceState& state, cudaStream_t stream) {
    const size_t smem = (static_cast<size_t>(per_block) * top_k + experts) * sizeof(int);
    auto kernel = blocks == 1 ? route_topk_kernel<V, true> : route_topk_kernel<V, false>;
    set_smem_limit_once(state, reinterpret_cast<const void*>(kernel), 200 * 1024, "cudaFuncSetAttribute(route smem)");
    const int threads = blocks > 1 || V > 8 ? kTopkThreads : 1024;
    launch_pdl(kernel, dim3(blocks), dim3(threads), smem, stream, "route_topk_kernel launch", logits, tokens, experts,
               ld, top_k, normalize, per_block, weights, ids, offsets, rows, slots, hist);
}

// 16 bytes of a row of Y as floats.
__device__ __forceinline__ void to_floats(const uint4& raw, float (&v)[8]) {
    const __half2* h = reinterpret_cast<const __half2*>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(h[i]);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void to_floats(const uint4& raw, float (&v)[4]) {
    v[0] = __uint_as_float(raw.x);
    v[1] = __uint_as_float(raw.y);
    v[2] = __uint_as_float(raw.z);
    v[3] = __uint_as_float(raw.w);
}

// out[t] = residual[t] + sum_j w_j y[slot_j], 16 bytes of columns a thread.  Bound by
// memory; the rows lie anywhere, so a thread asks for kBatch of them before it adds
// the first: 64.7 us for 16384 x 8 rows of 2 KB (6.0 TB/s), 76 us one at a time, 85
// us in batches of 8 (fewer threads resident).
constexpr int kBatch = 4;
template <class T>
__global__ void __launch_bounds__(256, 4) combine_kernel(const T* __restrict__ y, int64_t y_rows, int64_t ldy,
                                                      const int* __restrict__ slots, const float* __restrict__ weights,
                                                      int64_t tokens, int top_k, uint32_t per_row, const float* residual,
                                                      int64_t ldr, float* out, int64_t ldo) {
    constexpr int C = 16 / sizeof(T);
    pdl_wait();
    pdl_trigger();
    const int64_t units = tokens * per_row;
    for (int64_t u = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; u < units;
         u += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        const int64_t t = u / per_row, c = (u - t * per_row) * C;
        float4 r[C / 4];
#pragma unroll
        for (int i = 0; i < C / 4; ++i)
            r[i] = residual ? *reinterpret_cast<const float4*>(residual + t * ldr + c + 4 * i)
                            : make_float4(0.f, 0.f, 0.f, 0.f);
        float acc[C] = {};
        for (int j0 = 0; j0 < top_k; j0 += kBatch) {
            uint4 raw[kBatch];
            float w[kBatch];
            bool in[kBatch];
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
                const int slot = j0 + j < top_k ? __ldg(slots + t * top_k + j0 + j) : -1;
                in[j] = slot >= 0 && slot < y_rows;
                if (in[j]) raw[j] = __ldg(reinterpret_cast<const uint4*>(y + static_cast<int64_t>(slot) * ldy + c));
                w[j] = in[j] ? __ldg(weights + t * top_k + j0 + j) : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
                if (!in[j]) continue;
                float v[C];
                to_floats(raw[j], v);
#pragma unroll
                for (int i = 0; i < C; ++i) acc[i] = fmaf(w[j], v[i], acc[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < C / 4; ++i) {
            r[i].x += acc[4 * i];
            r[i].y += acc[4 * i + 1];
            r[i].z += acc[4 * i + 2];
            r[i].w += acc[4 * i + 3];
            *reinterpret_cast<float4*>(out + t * ldo + c + 4 * i) = r[i];
        }
    }
}

}  // namespace

size_t route_workspace_bytes(int64_t tokens, int experts, int top_k) {
    const int per_block = route_tokens_per_block(tokens, top_k);
    const int64_t blocks = (tokens + per_block - 1) / per_block;
    return blocks > 1 ? static_cast<size_t>(blocks + 1) * experts * sizeof(int) : 0;
}

void launch_route(const float* logits, int64_t tokens, int experts, int64_t ld, int top_k, int normalize,
                  float* weights, int32_t* ids, int32_t* offsets, int32_t* rows, int32_t* slots, void* workspace,
                  DeviceState& state, cudaStream_t stream) {
    const int per_block = route_tokens_per_block(tokens, top_k);
    const int blocks = static_cast<int>(std::max<int64_t>((tokens + per_block - 1) / per_block, 1));
    int* totals = static_cast<int*>(workspace);  // [experts], then the histograms [experts][blocks]
    int* hist = blocks > 1 ? totals + experts : nullptr;
    auto run = [&](auto width) {
        constexpr int V = decltype(width)::value;
        run_route<V>(logits, static_cast<int>(tokens), experts, ld, top_k, normalize, per_block, blocks, weights, ids,
                     offsets, rows, slots, hist, state, stream);
    };
    if (experts <= 64) run(std::integral_constant<int, 2>());
    else if (experts <= 128) run(std::integral_constant<int, 4>());
    else if (experts <= 256) run(std::integral_constant<int, 8>());
    else run(std::integral_constant<int, 32>());
    if (blocks == 1) return;
    launch_pdl(route_scan_kernel, dim3((experts + kPlaceThreads / 32 - 1) / (kPlaceThreads / 32)), dim3(kPlaceThreads),
               0, stream, "route_scan_kernel launch", hist, blocks, experts, totals);
    const int64_t items = tokens * top_k;
    launch_pdl(route_place_kernel, dim3(static_cast<unsigned>((items + kPlaceThreads - 1) / kPlaceThreads)),
               dim3(kPlaceThreads), experts * sizeof(int), stream, "route_place_kernel launch",
               static_cast<const int*>(hist), static_cast<const int*>(totals), items, experts, top_k, per_block, blocks,
               static_cast<const int*>(ids), offsets, rows, slots);
}

void launch_combine(const void* y, int y_type, int64_t y_rows, int64_t ldy, const int32_t* slots, const float* weights,
                    int64_t tokens, int top_k, int64_t width, const float* residual, int64_t ldr, float* out,
                    int64_t ldo, cudaStream_t stream) {
    const uint32_t per_row = static_cast<uint32_t>(width / (y_type == SAMQ_TYPE_F16 ? 8 : 4));
    const int64_t blocks = (tokens * per_row + 255) / 256;
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>(blocks, int64_t(1) << 24)));
    if (y_type == SAMQ_TYPE_F16)
        launch_pdl(combine_kernel<__half>, grid, dim3(256), 0, stream, "combine_kernel launch",
                   static_cast<const __half*>(y), y_rows, ldy, slots, weights, tokens, top_k, per_row, residual, ldr,
                   out, ldo);
    else
        launch_pdl(combine_kernel<float>, grid, dim3(256), 0, stream, "combine_kernel launch",
                   static_cast<const float*>(y), y_rows, ldy, slots, weights, tokens, top_k, per_row, residual, ldr,
                   out, ldo);
}

}  // namespace samq
