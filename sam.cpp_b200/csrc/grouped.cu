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

// The product's operand in plan order, f16 [rows][k]: row i is x[row_index ?
// row_index[i] : i], zeros for an index outside [0, x_rows) and for a row outside
// every group (which may hold anything: it is not read, so not reported either);
// f32 rows are staged by the Q8_1 rule on the way.  A thread moves 8 columns; four
// neighbouring threads a 32-value block.  Bound by memory: 2 + 2 (f16) or 4 + 2
// (f32) bytes an element.
template <class T, int U>
__global__ void __launch_bounds__(256) gather_rows_kernel(const T* __restrict__ x, int64_t x_rows, int64_t ldx,
                                                          const int* __restrict__ row_index,
                                                          const int* __restrict__ offsets, int groups, int64_t rows,
                                                          int k, __half* __restrict__ out, DeviceStatus* status) {
    pdl_wait();
    pdl_trigger();
    const int begin = __ldg(offsets), end = __ldg(offsets + groups);
    const uint32_t per_row = static_cast<uint32_t>(k / 8);
    const int64_t units = rows * per_row;
    const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
    // Whole warps: a unit's block neighbours are lanes of the same warp.  A thread asks for U units at once.
    for (int64_t u0 = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; u0 - (threadIdx.x & 31) < units;
         u0 += U * stride) {
        int64_t src[U];
        int c[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int64_t u = u0 + i * stride;
            const int64_t row = u < units ? u / per_row : 0;
            c[i] = static_cast<int>(u - row * per_row) * 8;
            src[i] = -1;
            if (u < units && row >= begin && row < end) src[i] = row_index ? __ldg(row_index + row) : row;
            if (src[i] >= x_rows) src[i] = -1;
        }
        constexpr int W = sizeof(T) == 2 ? 1 : 2;
        uint4 raw[U][W];
#pragma unroll
        for (int i = 0; i < U; ++i)
#pragma unroll
            for (int j = 0; j < W; ++j)
                raw[i][j] = src[i] >= 0 ? __ldg(reinterpret_cast<const uint4*>(x + src[i] * ldx + c[i]) + j)
                                        : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int64_t u = u0 + i * stride;
            uint4 o = raw[i][0];
            if constexpr (sizeof(T) == 4) {
                const float* f = reinterpret_cast<const float*>(raw[i]);
                const float v[8] = {f[0], f[1], f[2], f[3], f[4], f[5], f[6], f[7]};
                uint32_t pair[4];
                record_range(stage_q8_1<4, 8>(v, pair), status);
                o = make_uint4(pair[0], pair[1], pair[2], pair[3]);
            }
            if (u < units) *reinterpret_cast<uint4*>(out + u * 8) = o;
        }
    }
}

}  // namespace

void launch_gather_rows(const void* x, int x_type, int64_t x_rows, int64_t ldx, const int* row_index,
                        const int* offsets, int groups, int64_t rows, int k, __half* out, DeviceState& state,
                        cudaStream_t stream) {
    // Units per thread: several where there is work for the whole GPU all the same.
    const int64_t blocks = (rows * (k / 8) + 255) / 256;
    const bool many = blocks >= 16 * state.sm_count;
    const int64_t wanted = many ? (blocks + 3) / 4 : blocks;
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>(wanted, static_cast<int64_t>(state.sm_count) * 64)));
    const __half* xh = static_cast<const __half*>(x);
    const float* xf = static_cast<const float*>(x);
    if (x_type == SAMQ_TYPE_F16)
        launch_pdl(many ? gather_rows_kernel<__half, 4> : gather_rows_kernel<__half, 1>, grid, dim3(256), 0, stream,
                   "gather_rows_kernel launch", xh, x_rows, ldx, row_index, offsets, groups, rows, k, out,
                   state.status);
    else
        launch_pdl(many ? gather_rows_kernel<float, 4> : gather_rows_kernel<float, 1>, grid, dim3(256), 0, stream,
                   "gather_rows_kernel launch", xf, x_rows, ldx, row_index, offsets, groups, rows, k, out,
                   state.status);
}

// Few rows stream the packets, many take the f16 tiles.  Between, a call holds
// groups of either kind and only the device knows which: both kernels run and
// each leaves the other's groups alone.  From a mean of 64 rows on the tiles take
// small groups too, which are then few.  Tiles : both : packets alone, us, groups of
// equal size, 1024 -> 4096 Q4_K: 8 groups of 80 rows 18 : 20 : 28, of 64 17 : 20 : 17,
// of 48 18 : 18 : 16; 64 groups of 80 149 : 151 : 155, of 48 146 : 92 : 87.  The rule's
// worst case is many groups that all have just 64 rows: 64 such take 147 instead of 99
// (the f16 expansion of every group against its packets).
// With a mean of 16 rows or fewer the packet kernel does without the second launch as
// long as even all rows in one group would cost it no more than 96M decoded weights
// beyond one pass.  Packets alone : both, us, rows spread evenly and all in one group:
// 777 over 64 of 256 -> 2048 Q6_K 18 : 21 and 17 : 14; 256 over 32 of 1024 -> 4096 Q4_K
// 29 : 32 and 19 : 14; at the limit 384 over 32 30 : 33 and 26 : 17, 192 over 16 of
// 2048 -> 4096 Q8_0 35 : 37 and 24 : 19.  So it gains 3 us where groups are alike and
// loses at most 9 where they are not.
// With adapters the packet kernel also takes up to 256 rows of a narrow projection,
// whose few tiles would leave most SMs idle while it splits the depth.  Packets :
// tiles, us, 32 adapters of rank 24 and 4 of rank 16: 250 rows to n = 1024 17 : 23 and
// 11 : 13, to 1536 23 : 24 and 13 : 12, to 2560 25 : 22 and 11 : 12, to 4096 29 : 22 and
// 12 : 13; 100 rows to 2048 19 : 23 and 11 : 12, to 2560 25 : 23 and 14 : 13.  They meet
// between 40 and 64 units of 64 rows by 128 weight rows: hence 48.
RoutedPath routed_path(int64_t rows, int groups, int64_t n, int64_t k, bool adapted) {
    if (rows <= kRoutedFewRows) return RoutedPath::kRows;
    if (adapted && rows <= kRoutedFewAdapted && (rows + 63) / 64 * ((n + 127) / 128) <= 48) return RoutedPath::kRows;
    if (groups == 1 || rows >= int64_t(kRoutedFewRows) * groups) return RoutedPath::kTiles;
    if (rows <= int64_t(16) * groups && rows * n / 16 * k <= int64_t(96) << 20) return RoutedPath::kRows;
    return RoutedPath::kBoth;
}

void launch_routed(const RoutedProduct& p, DeviceState& state, cudaStream_t stream) {
    const RoutedPath path = routed_path(p.rows, p.groups, p.n, p.k, p.ids != nullptr);
    if (path != RoutedPath::kTiles)
        launch_routed_rows(p, path == RoutedPath::kRows ? INT_MAX : kRoutedFewRows, state, stream);
    if (path != RoutedPath::kRows)
        launch_routed_tile(p, path == RoutedPath::kTiles ? 1 : kRoutedFewRows + 1, state, stream);
}

}  // namespace samq
