// grouped.cu -- products whose weight depends on the row (samq_linear_grouped_v1,
// samq_linear_adapters_v1): y[i] = act(W_g x[row_index[i]] + bias_g + delta_i)
// for the rows i of group g, with delta the row's low-rank adapter.  Here the
// operand in plan order and the choice of kernel; the products themselves are in
// routed_rows.cu and routed_tile.cu, the adapters' down product in adapters.cu.
#include <algorithm>
#include <climits>

#include "samq_internal.hpp"

namespace samq {
namespace {

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

// Few rows stream the packets, many take the f16 tiles.  Between, a call holds
// groups of either kind and only the device knows which: both kernels run and
// each leaves the other's groups alone.
void launch_routed(const RoutedProduct& p, DeviceState& state, cudaStream_t stream) {
    const bool few = p.rows <= (p.ids ? kRoutedFewAdapted : kRoutedFewRows);
    const bool many = !few && (p.groups == 1 || p.rows >= 256 * p.groups);
    if (!many) launch_routed_rows(p, few ? INT_MAX : kRoutedFewRows, state, stream);
    if (!few) launch_routed_tile(p, many ? 1 : kRoutedFewRows + 1, state, stream);
}

}  // namespace samq
