// grouped.cu -- products whose weight depends on the row (samq_linear_grouped_v1,
// samq_linear_adapters_v1): y[i] = act(W_g x[row_index[i]] + bias_g + delta_i)
// for the rows i of group g, with delta the row's low-rank adapter.  Here the
// operand in plan order, the adapters' down product and the choice of kernel;
// the products themselves are in routed_rows.cu and routed_tile.cu.
#include <algorithm>
#include <climits>

#include "samq_internal.hpp"

namespace samq {
namespace {

// h2[i] = hi | lo of scale_a A_a x[i]: one warp per (row, rank index).
__global__ void __launch_bounds__(256) adapter_down_kernel(const RoutedProduct p, const __half* __restrict__ a_all,
                                                           const float* __restrict__ scales,
                                                           const int* __restrict__ ranks, __half* __restrict__ h2,
                                                           DeviceStatus* status) {
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const int64_t task = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
    const int64_t row = task / p.rank;
    const int r = static_cast<int>(task - row * p.rank);
    if (row >= p.rows) return;
    const int a = p.ids[row];
    float v = 0.0f;
    if (a >= 0 && a < p.adapter_count && r < ranks[a]) {
        const __half* av = a_all + (static_cast<int64_t>(a) * p.rank + r) * p.k;
        for (int c = lane; c < p.k; c += 32)
            v = fmaf(__half2float(p.x[row * p.ldx + c]), __half2float(av[c]), v);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        v *= scales[a];
    }
    record_range(!(fabsf(v) <= kOperandLimit), status);
    if (lane == 0) {
        const __half hi = __float2half_rn(v);
        h2[row * 2 * p.rank + r] = hi;
        h2[row * 2 * p.rank + p.rank + r] = __float2half_rn(v - __half2float(hi));
    }
}

// The product's operand in plan order, f16 [rows][k]: row i is x[row_index[i]]
// (zeros for an index outside [0, x_rows)), f32 rows staged by the Q8_1 rule on
// the way.  A thread moves 8 columns; four neighbouring threads a 32-value block.
// Bound by memory: 2 + 2 (f16) or 4 + 2 (f32) bytes an element.
template <class T>
__global__ void __launch_bounds__(256) gather_rows_kernel(const T* __restrict__ x, int64_t x_rows, int64_t ldx,
                                                          const int* __restrict__ row_index, int64_t rows, int k,
                                                          __half* __restrict__ out, DeviceStatus* status) {
    pdl_wait();
    pdl_trigger();
    const uint32_t per_row = static_cast<uint32_t>(k / 8);
    const int64_t units = rows * per_row;
    const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
    // Whole warps: a unit's block neighbours are lanes of the same warp.
    for (int64_t u = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; u - (threadIdx.x & 31) < units;
         u += stride) {
        const int64_t row = u < units ? u / per_row : 0;
        const int c = static_cast<int>(u - row * per_row) * 8;
        const int64_t src = u < units ? __ldg(row_index + row) : -1;
        const bool in = src >= 0 && src < x_rows;
        uint4 o = make_uint4(0, 0, 0, 0);
        if constexpr (sizeof(T) == 2) {
            if (in) o = __ldg(reinterpret_cast<const uint4*>(x + src * ldx + c));
        } else {
            float v[8] = {};
            if (in) {
                const float4 a = __ldg(reinterpret_cast<const float4*>(x + src * ldx + c));
                const float4 b = __ldg(reinterpret_cast<const float4*>(x + src * ldx + c) + 1);
                v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
                v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
            }
            uint32_t pair[4];
            record_range(stage_q8_1<4, 8>(v, pair), status);
            o = make_uint4(pair[0], pair[1], pair[2], pair[3]);
        }
        if (u < units) *reinterpret_cast<uint4*>(out + u * 8) = o;
    }
}

}  // namespace

void launch_gather_rows(const void* x, int x_type, int64_t x_rows, int64_t ldx, const int* row_index, int64_t rows,
                        int k, __half* out, DeviceState& state, cudaStream_t stream) {
    const int64_t blocks = (rows * (k / 8) + 255) / 256;
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>(blocks, static_cast<int64_t>(state.sm_count) * 32)));
    if (x_type == SAMQ_TYPE_F16)
        launch_pdl(gather_rows_kernel<__half>, grid, dim3(256), 0, stream, "gather_rows_kernel launch",
                   static_cast<const __half*>(x), x_rows, ldx, row_index, rows, k, out, state.status);
    else
        launch_pdl(gather_rows_kernel<float>, grid, dim3(256), 0, stream, "gather_rows_kernel launch",
                   static_cast<const float*>(x), x_rows, ldx, row_index, rows, k, out, state.status);
}

void launch_adapter_down(const RoutedProduct& p, const samq_adapters& ad, __half* h2, DeviceState& state,
                         cudaStream_t stream) {
    const int64_t warps = p.rows * ad.rank;
    launch_pdl(adapter_down_kernel, dim3(static_cast<unsigned>((warps + 7) / 8)), dim3(256), 0, stream,
               "adapter_down_kernel launch", p, static_cast<const __half*>(ad.a), static_cast<const float*>(ad.scale),
               static_cast<const int*>(ad.ranks), h2, state.status);
}

// Few rows stream the packets, many take the f16 tiles.  Between, a call holds
// groups of either kind and only the device knows which: both kernels run and
// each leaves the other's groups alone.
void launch_routed(const RoutedProduct& p, DeviceState& state, cudaStream_t stream) {
    const bool few = p.rows <= kRoutedFewRows;
    const bool many = !few && (p.groups == 1 || p.rows >= 256 * p.groups);
    if (!many) launch_routed_rows(p, few ? INT_MAX : kRoutedFewRows, state, stream);
    if (!few) launch_routed_tile(p, many ? 1 : kRoutedFewRows + 1, state, stream);
}

}  // namespace samq
