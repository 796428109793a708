// adapters.cu -- the down product of low-rank adapters: for every row i with
// adapter a = ids[i], h_i = scale_a A_a x_i (rank values, f32), stored as the f16
// pair hi | lo that routed_tile.cu multiplies as depth and routed_rows.cu adds up.
// x is the projection's operand (of f32 activations the staged one: one operand to
// read, and it is there).  The pair has h to 2^-22 |h| + 2^-25, as lo is subnormal
// below |h| = 2^-3; a scale of its own would have to be taken back in B, which has
// no bits to spare.
//
// Work is rank / n of the projection's, so this is a latency and L2 problem, not
// a tensor one: mma.sync m16n8k16 straight from global memory, no staging.  As a
// dot product does not care about the order of its depth, a lane's fragment takes
// eight consecutive columns (one 16-byte load of x, one of A_a, the same columns),
// which serve two instructions, and the four lanes of a row read 64 bytes together.
// A window of rows is cut into tasks of up to 32 rows of one adapter, in rising
// order of the adapters; a block takes every gridDim.y-th task of a window, RANK of
// the rank at a time (block layer z the z-th, z + gridDim.z-th ... such).  Its warps
// split the depth and add their sums in shared memory in warp order.  (Tasks from
// windows of 32 rows read A_a once for every few rows of a mixed batch: 33 us for 4000
// rows of 24 adapters, rank 16, 70 us for 2000, rank 128, from windows of 256 24 and
// 35.)  Few rows are a chain of latencies, which a larger window only lengthens (16
// rows: 11.1 us with the product, 12.0 from 256): windows of 32, and up to 64 rows 16
// warps, 16 of the rank a block.  Many rows are throughput: 8 warps, 32 of the rank,
// two blocks an SM (5184 rows, rank 64: 6 us more with the product the other way
// round; two or four steps of the depth in flight a warp: 1.5 to 2.5 us more).
// The pair of a row without adapter is not written, as nothing reads it.
#include <algorithm>

#include "samq_internal.hpp"

namespace samq {
namespace {

constexpr int kRows = 32;  // of a task

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

template <int WARPS, int RANK, int WINDOW>
__global__ void __launch_bounds__(32 * WARPS)
adapter_down_kernel(const RoutedProduct p, const __half* __restrict__ a_all, const float* __restrict__ scales,
                    const int* __restrict__ ranks, __half* __restrict__ h2, DeviceStatus* status) {
    __shared__ float part[WARPS][kRows][RANK + 1];
    __shared__ int lists[WARPS][kRows];  // every warp's copy of the task's rows
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row0 = blockIdx.x * WINDOW;
    pdl_wait();
    pdl_trigger();
    int id[WINDOW / 32];  // of rows row0 + 32 j + lane
#pragma unroll
    for (int j = 0; j < WINDOW / 32; ++j) {
        const int64_t row = row0 + 32 * j + lane;
        id[j] = row < p.rows ? __ldg(p.ids + row) : -1;
        if (id[j] >= p.adapter_count) id[j] = -1;
    }
    const int q = lane & 3, g = lane >> 2;  // 8-column group, row of the fragment
    int* list = lists[warp];
    int a = -1, found = 0, start = 0;  // the adapter, its rows in the window, the first of the next task
    for (int task = 0;; ++task) {
        if (start >= found) {
            // The next larger adapter of these rows.
            int next = p.adapter_count;
#pragma unroll
            for (int j = 0; j < WINDOW / 32; ++j)
                if (id[j] > a) next = min(next, id[j]);
            a = __reduce_min_sync(0xffffffffu, next);
            if (a >= p.adapter_count) break;
            found = start = 0;
#pragma unroll
            for (int j = 0; j < WINDOW / 32; ++j) found += __popc(__ballot_sync(0xffffffffu, id[j] == a));
        }
        const int first = start;
        start += kRows;
        if (task % static_cast<int>(gridDim.y) != static_cast<int>(blockIdx.y)) continue;
        const int count = min(kRows, found - first);
        const int used = __ldg(ranks + a);
        const float scale = __ldg(scales + a);
        __syncthreads();  // the previous task's lists and sums have been read
        int before = 0;
#pragma unroll
        for (int j = 0; j < WINDOW / 32; ++j) {
            const unsigned in = __ballot_sync(0xffffffffu, id[j] == a);
            const int at = before + __popc(in & ((1u << lane) - 1u)) - first;
            if (id[j] == a && at >= 0 && at < kRows) list[at] = row0 + 32 * j + lane;
            before += __popc(in);
        }
        __syncwarp();
        const __half* xr[4];  // the fragment's rows g + 8 i
#pragma unroll
        for (int i = 0; i < 4; ++i)
            xr[i] = g + 8 * i < count ? p.x + static_cast<int64_t>(list[g + 8 * i]) * p.ldx + 8 * q : nullptr;
        for (int c0 = static_cast<int>(blockIdx.z) * RANK; c0 < p.rank; c0 += static_cast<int>(gridDim.z) * RANK) {
            float acc[2][RANK / 8][4] = {};
            if (c0 < used) {
                const __half* aa = a_all + (static_cast<int64_t>(a) * p.rank + c0 + g) * p.k + 8 * q;
                for (int k = 32 * warp; k < p.k; k += 32 * WARPS) {
                    uint4 x[4], b[RANK / 8];
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = load16(xr[i] + k, xr[i] != nullptr);
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
                if (r < count && c0 + c < p.rank) {
#pragma unroll
                    for (int w = 0; w < WARPS; ++w) v += part[w][r][c];
                    v = c0 + c < used ? v * scale : 0.0f;
                    const __half hi = __float2half_rn(v);
                    __half* out = h2 + static_cast<int64_t>(list[r]) * 2 * p.rank + c0 + c;
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
    const __half* a = ad.a;
    const float* scale = ad.scale;
    const int* ranks = ad.ranks;
    auto run = [&](auto kernel, int threads, int window, int layers) {
        const int windows = static_cast<int>((p.rows + window - 1) / window);
        // Blocks of a window: as many as it may have tasks, while they fill the GPU four times at most.
        const int most = std::min({window / kRows + ad.count, window, static_cast<int>(p.rows)});
        const int columns = std::max(1, std::min(most, 4 * state.sm_count / windows));
        launch_pdl(kernel, dim3(windows, columns, layers), dim3(threads), 0, stream, "adapter_down_kernel launch", p, a,
                   scale, ranks, h2, state.status);
    };
    if (p.rows <= 64) run(adapter_down_kernel<16, 16, 32>, 512, 32, p.rank / 16);
    else if (p.rows <= 256) run(adapter_down_kernel<8, 32, 32>, 256, 32, 1);
    else run(adapter_down_kernel<8, 32, 256>, 256, 256, 1);
}

}  // namespace samq
