// adapters.cu -- the down product of low-rank adapters: for every row i with
// adapter a = ids[i], h_i = scale_a A_a x_i (rank values, f32), stored as the f16
// pair hi | lo that routed_tile.cu multiplies as depth and routed_rows.cu adds up.
//
// Work is rank / n of the projection's, so this is a latency and L2 problem, not
// a tensor one: mma.sync m16n8k16 straight from global memory, no staging.  As a
// dot product does not care about the order of its depth, a lane's fragment takes
// eight consecutive columns (one 16-byte load of x, one of A_a, the same columns),
// which serve two instructions, and the four lanes of a row read 64 bytes together.
// A block takes 32 rows, RANK of the rank at a time (block layer z the z-th, z +
// gridDim.z-th ... such) and one adapter of the several its rows may name (block
// column y likewise, in rising order); its warps split the depth and add their sums
// in shared memory in warp order.  Few rows are a chain of latencies: 16 warps, 16 of
// the rank a block (16 rows with an adapter each, k = 1024: 12.0 -> 11.4 us with the
// product).  Many rows are throughput: 8 warps, 32 of the rank, three blocks an SM
// (5184 rows, rank 64: 76 us the other way round against 70).  The pair of a row
// without adapter is not written, as nothing reads it.
#include <algorithm>

#include "samq_internal.hpp"

namespace samq {
namespace {

constexpr int kRows = 32;

__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
        "%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 load16(const __half* p, bool in) {
    return in ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0);
}

template <int WARPS, int RANK>
__global__ void __launch_bounds__(32 * WARPS)
adapter_down_kernel(const RoutedProduct p, const __half* __restrict__ a_all, const float* __restrict__ scales,
                    const int* __restrict__ ranks, __half* __restrict__ h2, DeviceStatus* status) {
    __shared__ float part[WARPS][kRows][RANK + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row0 = blockIdx.x * kRows;
    pdl_wait();
    pdl_trigger();
    const int rows = min(kRows, static_cast<int>(p.rows) - row0);
    int id = lane < rows ? __ldg(p.ids + row0 + lane) : -1;
    if (id >= p.adapter_count) id = -1;
    const int q = lane & 3, g = lane >> 2;  // 8-column group, row of the fragment
    int last = -1;
    for (int index = 0;; ++index) {
        // The next larger adapter of these rows.
        const int a = __reduce_min_sync(0xffffffffu, id > last ? id : p.adapter_count);
        if (a >= p.adapter_count) break;
        last = a;
        if (index % static_cast<int>(gridDim.y) != static_cast<int>(blockIdx.y)) continue;
        const int used = __ldg(ranks + a);
        const float scale = __ldg(scales + a);
        const unsigned members = __ballot_sync(0xffffffffu, id == a);
        for (int c0 = static_cast<int>(blockIdx.z) * RANK; c0 < p.rank; c0 += static_cast<int>(gridDim.z) * RANK) {
            float acc[2][RANK / 8][4] = {};
            if (c0 < used) {
                const __half* aa = a_all + (static_cast<int64_t>(a) * p.rank + c0 + g) * p.k + 8 * q;
                const __half* xr = p.x + static_cast<int64_t>(row0 + g) * p.ldx + 8 * q;
                for (int k = 32 * warp; k < p.k; k += 32 * WARPS) {
                    uint4 x[4], b[RANK / 8];
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = load16(xr + 8 * i * p.ldx + k, (members >> (g + 8 * i)) & 1u);
#pragma unroll
                    for (int i = 0; i < RANK / 8; ++i)
                        b[i] = load16(aa + static_cast<int64_t>(8 * i) * p.k + k, c0 + 8 * i < used);
#pragma unroll
                    for (int i = 0; i < RANK / 8; ++i)
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            mma_16816(acc[m][i], x[2 * m].x, x[2 * m + 1].x, x[2 * m].y, x[2 * m + 1].y, b[i].x, b[i].y);
                            mma_16816(acc[m][i], x[2 * m].z, x[2 * m + 1].z, x[2 * m].w, x[2 * m + 1].w, b[i].z, b[i].w);
                        }
                }
            }
            __syncthreads();  // the previous sums have been read
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int i = 0; i < RANK / 8; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        part[warp][16 * m + g + 8 * (j >> 1)][8 * i + 2 * q + (j & 1)] = acc[m][i][j];
            __syncthreads();
            for (int i = threadIdx.x; i < kRows * RANK; i += 32 * WARPS) {
                const int r = i / RANK, c = i % RANK;
                float v = 0.0f;
                if (((members >> r) & 1u) && c0 + c < p.rank) {
#pragma unroll
                    for (int w = 0; w < WARPS; ++w) v += part[w][r][c];
                    v = c0 + c < used ? v * scale : 0.0f;
                    const __half hi = __float2half_rn(v);
                    __half* out = h2 + static_cast<int64_t>(row0 + r) * 2 * p.rank + c0 + c;
                    out[0] = hi;
                    out[p.rank] = __float2half_rn(v - __half2float(hi));
                }
                record_range(!(fabsf(v) <= kOperandLimit), status);
            }
        }
    }
}

}  // namespace

void launch_adapter_down(const RoutedProduct& p, const samq_adapters& ad, __half* h2, DeviceState& state,
                         cudaStream_t stream) {
    const int tiles = static_cast<int>((p.rows + kRows - 1) / kRows);
    // Few rows may name an adapter each: a block apiece.  Many rows fill the GPU by themselves.
    const bool few = p.rows <= 64;
    const int columns = std::max(1, std::min({ad.count, kRows, 4 * state.sm_count / tiles}));
    const __half* a = ad.a;
    const float* scale = ad.scale;
    const int* ranks = ad.ranks;
    if (few)
        launch_pdl(adapter_down_kernel<16, 16>, dim3(tiles, columns, p.rank / 16), dim3(512), 0, stream,
                   "adapter_down_kernel launch", p, a, scale, ranks, h2, state.status);
    else
        launch_pdl(adapter_down_kernel<8, 32>, dim3(tiles, columns), dim3(256), 0, stream,
                   "adapter_down_kernel launch", p, a, scale, ranks, h2, state.status);
}

}  // namespace samq
