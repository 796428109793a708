// routed_tile.cu -- the routed product for groups of many rows, on the tensor
// cores: y[i] = act(W_g x[row_index[i]] + bias_g + delta_i) over tiles of 128 (or
// 256, a CTA pair) consecutive plan rows of one group by BN weight rows.
//
// Mathematics.  One tile is D = X_tile . W_tile^T over k, in f32 in TMEM.  The
// adapters ride on the same accumulator as more depth:
//   delta_i = B_a h_i, h_i = scale_a A_a x_i (a = ids[i]),
//   D += [hi(H) | lo(H)] . [B_a | B_a]^T for every adapter a with rows in the tile,
// on the accumulator rows i with ids[i] == a alone: the MMA leaves the lanes of the
// others as they are.  The pair keeps h to 2^-22 |h| + 2^-25: f32's level against the
// f16 rounding of B, until lo becomes subnormal below |h| = 2^-3.  (Zeroing the other rows of the left factor by a TMA row gather
// instead made such a step 1.2 us, three times a step of W.)
//
// x arrives in plan order: a row_index has been applied by gather_rows_kernel.
// Gathering inside this kernel was measured and not kept (10368 rows of 8
// experts, 1024 -> 4736, without GELU; then 107 us in plan order, 8 us for the copy):
// x by the row gather of TMA 287 us, by 16-byte asynchronous copies of four
// warps 272 us (213 us when no row was to be read: the hand-over of each step to
// the tensor core bounds it, not the memory).
//
// Pipeline (one CTA or CTA pair per SM or TPC, persistent over the tiles of all
// groups):
//   warp 0     W producer: BN (a pair: BN / 2 each) x 64 of W per step by TMA,
//              128-byte swizzle, kStages deep;
//   last warp  X producer: 128 x 64 of X.  Each step's `last` flag travels with its
//              stage, as only the producers know how many adapters a tile has.  Two
//              warps as a step's wait, announcement and two copies take one thread
//              longer than the tensor cores need for it (512 cycles);
//   warp 1     TMEM owner; one thread (of the even CTA) issues tcgen05.mma;
//   warps 2..  epilogue: accumulator out of TMEM, bias, erf-GELU, 32 rows of 128
//              bytes at a time through swizzled shared memory: one TMA store, or,
//              where the group ends inside them, coalesced stores of its own rows.
//              The next tile's MMAs overlap it.
// Measured (10368 rows of 8 experts, 1024 -> 4736): 99 us, 1.01 PFLOP/s, 116 with the
// row copy and GELU.  In the kernel the tensor pipe is busy 55% of the time, the issue
// slots 33%, the HBM 17%: a step's 32 KB an SM from L2 and the board's power bound it.
// Staging half of f32 rows beside the other half's product was measured and not kept
// (4736 -> 1024): they overlap, but slow each other down by as much as is saved.
// Every wait is bounded.  No load uses multicast.
#include <algorithm>

#include "samq_internal.hpp"

namespace samq {
namespace {

constexpr int BM = 128;  // rows of a CTA's tile
constexpr int BK = 64;   // depth of a step: one 128-byte swizzle row of f16
constexpr int kAccStride = 256;
constexpr int kEpilogueWarps = 8;
constexpr int kThreads = 96 + 32 * kEpilogueWarps;
constexpr int kXWarp = 2 + kEpilogueWarps;
constexpr int kSlabBytes = 32 * 128;  // an epilogue warp's staging: 32 rows of 128 bytes
constexpr int kSmemLimit = 232448;

// GROUPS: the most groups the tables hold.  They take a stage's room only in the
// instance for many groups: six stages against five are 151 us against 158 for 10368
// staged rows of 8 groups, 4736 -> 1024.
template <int CTAS, int BN, int GROUPS>
struct TileSmem {
    static constexpr int a_bytes = BM * BK * 2;
    static constexpr int b_bytes = BN / CTAS * BK * 2;
    static constexpr int stage = a_bytes + b_bytes;
    static constexpr int out = kEpilogueWarps * kSlabBytes;
    static constexpr int tables = (3 * GROUPS + 1) * 4;  // begin, end, tile prefix of each group
    static constexpr int fixed = 1024 + out + tables + 384;
    static constexpr int stages = (kSmemLimit - fixed) / stage > 8 ? 8 : (kSmemLimit - fixed) / stage;
    static constexpr int b_off = stages * a_bytes;
    static constexpr int out_off = stages * stage;
    static constexpr int bar_off = out_off + out;
    static constexpr int table_off = bar_off + 384;
    static constexpr int total = stages * stage + fixed;
};

struct TileMaps {
    CUtensorMap x;       // box 64 x 128
    CUtensorMap w;       // box 64 x BN / CTAS
    CUtensorMap h;       // adapters: [rows][2 rank], box 64 x 128
    CUtensorMap b;       // adapters: [adapters * n][2 rank], box 64 x BN / CTAS
    CUtensorMap y;       // output, box 128 bytes x 32
};

template <int CTAS>
__device__ __forceinline__ void tma_tile(void* dst, const CUtensorMap* map, uint64_t* local, uint32_t bar, int x,
                                         int y) {
    if constexpr (CTAS == 1) tma_load_2d(dst, map, local, x, y);
    else tma_load_2d_pair(dst, map, bar, x, y);
}

__device__ __forceinline__ int clamp_row(int v, int64_t rows) {
    return v < 0 ? 0 : v > rows ? static_cast<int>(rows) : v;
}

struct Tile {
    int group, row0, end, col0;  // plan rows row0 .. end - 1, columns col0 ..
    bool narrow;                 // half the tile's columns or fewer: half the MMA
};

// The groups' tiles in order: s_first[g] is the number of row tiles before group g.
__device__ __forceinline__ Tile find_tile(int tile, int n_tiles, int n, int bn, int rows_per_tile, int groups,
                                          const int* s_first, const int* s_begin, const int* s_end) {
    const int rt = tile / n_tiles;
    int lo = 0, hi = groups;  // s_first[lo] <= rt < s_first[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_first[mid] <= rt) lo = mid;
        else hi = mid;
    }
    Tile t;
    t.group = lo;
    t.row0 = s_begin[lo] + (rt - s_first[lo]) * rows_per_tile;
    t.end = s_end[lo];
    t.col0 = (tile - rt * n_tiles) * bn;
    t.narrow = n - t.col0 <= bn / 2;
    return t;
}

template <int CTAS, int BN, int GROUPS>
__global__ void __launch_bounds__(kThreads, 1)
routed_tile_kernel(const __grid_constant__ TileMaps maps, const RoutedProduct p, int min_rows, DeviceStatus* status) {
    using L = TileSmem<CTAS, BN, GROUPS>;
    constexpr int kStages = L::stages;
    static_assert(kStages >= 3 && L::total <= kSmemLimit, "shared memory budget");
    static_assert(2 * 8 * kStages + 5 * 8 + 8 + 36 * kStages <= 384, "barrier space");
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sa = smem;
    uint8_t* sb = smem + L::b_off;
    int* s_begin = reinterpret_cast<int*>(smem + L::table_off);
    int* s_end = s_begin + GROUPS;
    int* s_first = s_end + GROUPS;
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::bar_off);
    uint64_t* empty = full + kStages;
    uint64_t* tfull = empty + kStages;
    uint64_t* tempty = tfull + 2;
    uint64_t* drain = tempty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    // Of each stage: kLast | kMasked, and the accumulator lanes an adapter step leaves alone.
    constexpr int kLast = 1, kMasked = 2;
    volatile int* step_kind = reinterpret_cast<int*>(tmem_slot + 2);
    volatile uint32_t* step_off = tmem_slot + 2 + kStages;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = CTAS == 2 ? static_cast<int>(cluster_cta_rank()) : 0;
    const int unit = blockIdx.x / CTAS, units = gridDim.x / CTAS;
    constexpr int kTileRows = CTAS * BM;
    const int n_tiles = (p.n + BN - 1) / BN;
    const int kblocks = (p.k + BK - 1) / BK;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&tfull[b], 1);
            mbar_init(&tempty[b], CTAS * kEpilogueWarps);
        }
        mbar_init(drain, 1);
        fence_barrier_init();
        tma_prefetch_desc(&maps.x);
        tma_prefetch_desc(&maps.w);
        tma_prefetch_desc(&maps.y);
    }
    if (warp == 1) {
        if constexpr (CTAS == 2) tmem_alloc_pair(tmem_slot, 2 * kAccStride);
        else tmem_alloc(tmem_slot, 2 * kAccStride);
    }
    // What the previous kernel may write is read from here on.  With adapters that
    // kernel is the down product, which began its own work only after everything
    // before it had completed: all but its pairs may be read at once, and the X
    // producer waits for those.
    if (!p.ids) pdl_wait();
    if (warp == 2) {
        int carry = 0;
        for (int base = 0; base < p.groups; base += 32) {
            const int g = base + lane;
            int begin = 0, end = 0, tiles = 0;
            if (g < p.groups) {
                begin = p.offsets ? clamp_row(__ldg(p.offsets + g), p.rows) : 0;
                end = p.offsets ? max(begin, clamp_row(__ldg(p.offsets + g + 1), p.rows)) : static_cast<int>(p.rows);
                tiles = end - begin >= min_rows ? (end - begin + kTileRows - 1) / kTileRows : 0;
                s_begin[g] = begin;
                s_end[g] = end;
            }
            int sum = tiles;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += u;
            }
            if (g < p.groups) s_first[g] = carry + sum - tiles;
            carry += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (lane == 0) s_first[p.groups] = carry;
    }
    tc_fence_before();
    if constexpr (CTAS == 2) cluster_sync_all();
    else __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int tiles = s_first[p.groups] * n_tiles;

    if (warp == 0 || warp == kXWarp) {
        // Both producers walk the same steps; the X warp announces them.
        const bool is_x = warp == kXWarp;
        int s = 0;
        uint32_t ph = 0;
        uint32_t issued = 0, issued_phase = 0;
        bool ok = true;
        const uint32_t full_bar = CTAS == 2 ? cluster_map(full, 0) : smem_u32(full);  // the even CTA's
        // The whole warp waits for the next stage; one thread of the X warp announces the step.
        auto open = [&](int kind, const uint32_t* off) -> bool {
            if (!mbar_wait_warp(&empty[s], ph ^ 1u, status, 61)) return false;
            if (is_x && rank == 0 && elect_one()) {
                step_kind[s] = kind;
                if (kind & kMasked) {
#pragma unroll
                    for (int j = 0; j < 4 * CTAS; ++j) step_off[8 * s + j] = off[j];
                }
                mbar_arrive_expect_tx(&full[s], CTAS * L::stage);
            }
            __syncwarp();
            issued |= 1u << s;
            issued_phase = (issued_phase & ~(1u << s)) | (ph << s);
            return true;
        };
        auto advance = [&] {
            if (++s == kStages) {
                s = 0;
                ph ^= 1u;
            }
        };
        for (int tile = unit; tile < tiles && ok; tile += units) {
            const Tile t = find_tile(tile, n_tiles, p.n, BN, kTileRows, p.groups, s_first, s_begin, s_end);
            const int row0 = t.row0 + rank * BM;
            const int b_half = rank * (t.narrow ? BN / 2 : BN) / CTAS;
            // The adapters of the tile's rows (a pair's 256 for both CTAs): rows 32 j + lane.
            int id[4 * CTAS];
            int next = p.adapter_count;
            if (p.ids) {
#pragma unroll
                for (int j = 0; j < 4 * CTAS; ++j) {
                    const int row = t.row0 + 32 * j + lane;
                    id[j] = row < t.end ? __ldg(p.ids + row) : -1;
                    if (id[j] >= 0) next = min(next, id[j]);
                }
                next = __reduce_min_sync(0xffffffffu, next);
            }
            const int wrow = t.group * p.n + t.col0 + b_half;
            const bool plain = next >= p.adapter_count;
            for (int kb = 0; kb < kblocks; ++kb) {
                ok = open(kb == kblocks - 1 && plain ? kLast : 0, nullptr);
                if (!ok) break;
                if (elect_one()) {
                    if (is_x)
                        tma_tile<CTAS>(sa + s * L::a_bytes, &maps.x, &full[s], full_bar + 8 * s, kb * BK, row0);
                    else
                        tma_tile<CTAS>(sb + s * L::b_bytes, &maps.w, &full[s], full_bar + 8 * s, kb * BK, wrow);
                }
                __syncwarp();
                advance();
            }
            if (!p.ids) continue;
            if (is_x && ok && next < p.adapter_count) pdl_wait();
            while (ok && next < p.adapter_count) {
                const int a = next;
                next = p.adapter_count;
                uint32_t off[4 * CTAS];
#pragma unroll
                for (int j = 0; j < 4 * CTAS; ++j) {
                    off[j] = ~__ballot_sync(0xffffffffu, id[j] == a);
                    if (id[j] > a) next = min(next, id[j]);
                }
                next = __reduce_min_sync(0xffffffffu, next);
                for (int c = 0; c < 2 * p.rank && ok; c += BK) {
                    ok = open(kMasked | (c + BK >= 2 * p.rank && next >= p.adapter_count ? kLast : 0), off);
                    if (!ok) break;
                    if (elect_one()) {
                        if (is_x)
                            tma_tile<CTAS>(sa + s * L::a_bytes, &maps.h, &full[s], full_bar + 8 * s, c, row0);
                        else
                            tma_tile<CTAS>(sb + s * L::b_bytes, &maps.b, &full[s], full_bar + 8 * s, c,
                                           a * p.n + t.col0 + b_half);
                    }
                    __syncwarp();
                    advance();
                }
            }
        }
        if (is_x) pdl_wait();  // if not before: the kernel ends after its predecessors
        pdl_trigger();         // all of this warp's loads are issued
        if (!ok && lane == 0) {
            // Let the copies in flight land before the CTA exits.
            if constexpr (CTAS == 1) {
                for (int i = 0; i < kStages; ++i)
                    if (issued & (1u << i)) mbar_wait(&full[i], (issued_phase >> i) & 1u, status, 65);
            } else {
                const uint64_t start = global_timer_ns();
                while (global_timer_ns() - start < 2000000ull) __nanosleep(1000);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0 && elect_one()) {
            constexpr uint32_t idesc_full = idesc_f16_f32(CTAS * BM, BN), idesc_half = idesc_f16_f32(CTAS * BM, BN / 2);
            // Descriptors of stage 0; a stage or 32 bytes on only moves the address field (16-byte units).
            const uint64_t a_desc = smem_desc_sw128(smem_u32(sa)), b_desc = smem_desc_sw128(smem_u32(sb));
            int s = 0;
            uint32_t ph = 0;
            auto wait_full = [&](int i, uint32_t phase) {
                return CTAS == 2 ? mbar_wait_cluster(&full[i], phase, status, 63) : mbar_wait(&full[i], phase, status, 63);
            };
            auto probe_full = [&](int i, uint32_t phase) {
                return CTAS == 2 ? mbar_test_wait_cluster(&full[i], phase) : mbar_test_wait(&full[i], phase);
            };
            bool ready = false;
            int piece = 0;  // first column of the next adapter step's piece of the pair
            int acc = 0;
            uint32_t acc_ph = 0;
            bool ok = true;
            for (int tile = unit; tile < tiles && ok; tile += units) {
                const bool free = CTAS == 2 ? mbar_wait_cluster(&tempty[acc], acc_ph ^ 1u, status, 62)
                                            : mbar_wait(&tempty[acc], acc_ph ^ 1u, status, 62);
                if (!free) break;
                tc_fence_after();
                const uint32_t d = tmem_base + static_cast<uint32_t>(acc * kAccStride);
                const uint32_t idesc = p.n - tile % n_tiles * BN <= BN / 2 ? idesc_half : idesc_full;
                uint32_t accumulate = 0;
                bool last = false;
                while (!last) {
                    // The probe of this stage was issued under the previous step's MMAs.
                    if (!ready && !wait_full(s, ph)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const int kind = step_kind[s];
                    last = kind & kLast;
                    uint32_t off[4 * CTAS] = {};
                    if (kind & kMasked) {
#pragma unroll
                        for (int j = 0; j < 4 * CTAS; ++j) off[j] = step_off[8 * s + j];
                    }
                    const uint64_t ad = a_desc + static_cast<uint32_t>(s * (L::a_bytes >> 4));
                    const uint64_t bd = b_desc + static_cast<uint32_t>(s * (L::b_bytes >> 4));
                    const int now = s;
                    if (++s == kStages) {
                        s = 0;
                        ph ^= 1u;
                    }
                    ready = probe_full(s, ph);
                    if (kind & kMasked) {
                        // The last piece of a pair may be short of 64 columns.
                        const int deep = min(BK, 2 * p.rank - piece);
                        piece = piece + BK < 2 * p.rank ? piece + BK : 0;
#pragma unroll
                        for (int kk = 0; kk < BK / 16; ++kk) {
                            if (16 * kk >= deep) break;
                            if constexpr (CTAS == 2) tc_mma_f16_pair_lanes(d, ad + 2 * kk, bd + 2 * kk, idesc, off);
                            else tc_mma_f16_lanes(d, ad + 2 * kk, bd + 2 * kk, idesc, off);
                        }
                    } else {
#pragma unroll
                        for (int kk = 0; kk < BK / 16; ++kk) {
                            if constexpr (CTAS == 2) tc_mma_f16_pair(d, ad + 2 * kk, bd + 2 * kk, idesc, accumulate);
                            else tc_mma_f16(d, ad + 2 * kk, bd + 2 * kk, idesc, accumulate);
                            accumulate = 1;
                        }
                    }
                    if constexpr (CTAS == 2) tc_commit_both(&empty[now]);
                    else tc_commit(&empty[now]);
                }
                if (!ok) break;
                if constexpr (CTAS == 2) tc_commit_both(&tfull[acc]);
                else tc_commit(&tfull[acc]);
                acc ^= 1;
                if (acc == 0) acc_ph ^= 1u;
            }
            // Every MMA this thread issued is complete before TMEM is released.
            if constexpr (CTAS == 2) tc_commit_pair(cluster_map(drain, 0));
            else tc_commit(drain);
            mbar_wait(drain, 0, status, 66);
        }
        __syncwarp();
    } else {
        constexpr int kShare = BN / (kEpilogueWarps / 4);  // columns of a warp
        const int quarter = warp & 3;                      // TMEM lanes 32 * quarter ..
        const int part = (warp - 2) >> 2;
        const bool f16 = p.y_type == SAMQ_TYPE_F16;
        const int elem = f16 ? 2 : 4;
        const int slab_cols = 128 / elem;
        uint8_t* slab = smem + L::out_off + (warp - 2) * kSlabBytes;
        int acc = 0;
        uint32_t acc_ph = 0;
        for (int tile = unit; tile < tiles; tile += units) {
            const Tile t = find_tile(tile, n_tiles, p.n, BN, kTileRows, p.groups, s_first, s_begin, s_end);
            const int row0 = t.row0 + rank * BM + quarter * 32;
            const float* bias = p.bias ? p.bias + static_cast<int64_t>(t.group) * p.n + t.col0 : nullptr;
            const bool bias_vec = (reinterpret_cast<uintptr_t>(bias) & 15u) == 0;
            // Warp-uniform: the TMEM loads below are warp-collective.
            if (!mbar_wait_warp(&tfull[acc], acc_ph, status, 64)) break;
            tc_fence_after();
#pragma unroll 1
            for (int c0 = part * kShare; c0 < (part + 1) * kShare; c0 += slab_cols) {
                const int inside = p.n - t.col0 - c0;  // columns from here to the group's last
                if (inside <= 0 || row0 >= t.end) break;
                if (lane == 0) bulk_wait_group_read<0>();  // the slab's last store has left it
                __syncwarp();
#pragma unroll 1
                for (int c = c0; c < c0 + slab_cols; c += 32) {
                    const int left = p.n - t.col0 - c;
                    uint32_t r[32];
                    tc_ld_32x32b_x32(tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) +
                                         static_cast<uint32_t>(acc * kAccStride + c),
                                     r);
                    float v[32];
                    if (bias && left >= 32 && bias_vec) {
                        const float4* b4 = reinterpret_cast<const float4*>(bias + c);
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float4 b = __ldg(b4 + j);
                            v[4 * j] = b.x; v[4 * j + 1] = b.y; v[4 * j + 2] = b.z; v[4 * j + 3] = b.w;
                        }
                    } else {
                        const float mine = bias && lane < left ? __ldg(bias + c + lane) : 0.0f;
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = __shfl_sync(0xffffffffu, mine, i);
                    }
                    tc_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] += __uint_as_float(r[i]);
                    if (p.gelu) {
#pragma unroll
                        for (int i = 0; i < 32; i += 2) gelu_erf2(v[i], v[i + 1]);
                    }
                    // 16-byte unit u of row `lane` at u ^ (lane % 8): the store's 128-byte swizzle.
                    if (f16) {
                        const int u0 = (c - c0) >> 3;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            uint32_t o[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const __half2 h = __floats2half2_rn(v[8 * j + 2 * i], v[8 * j + 2 * i + 1]);
                                o[i] = *reinterpret_cast<const uint32_t*>(&h);
                            }
                            *reinterpret_cast<uint4*>(slab + lane * 128 + (((u0 + j) ^ (lane & 7)) << 4)) =
                                make_uint4(o[0], o[1], o[2], o[3]);
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            *reinterpret_cast<float4*>(slab + lane * 128 + ((j ^ (lane & 7)) << 4)) =
                                make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                    }
                }
                if (row0 + 32 <= t.end) {
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        tma_store_2d(&maps.y, slab, t.col0 + c0, row0);  // clipped at column n
                        bulk_commit_group();
                    }
                } else {
                    // Another group's rows (or the caller's) follow: 8 lanes a row, the group's own rows only.
                    __syncwarp();
                    const int u = lane & 7, units_inside = min(inside, slab_cols) * elem / 16;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int rr = 4 * i + (lane >> 3);
                        if (row0 + rr >= t.end) continue;
                        const uint8_t* from = slab + rr * 128 + ((u ^ (rr & 7)) << 4);
                        uint8_t* to = static_cast<uint8_t*>(p.y) +
                                      (static_cast<int64_t>(row0 + rr) * p.ldy + t.col0 + c0) * elem + 16 * u;
                        if (u < units_inside) {
                            *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(from);
                        } else if (u == units_inside) {
                            for (int b = 0; b < (inside * elem) % 16 && inside < slab_cols; b += elem) {
                                if (f16) *reinterpret_cast<__half*>(to + b) = *reinterpret_cast<const __half*>(from + b);
                                else *reinterpret_cast<float*>(to + b) = *reinterpret_cast<const float*>(from + b);
                            }
                        }
                    }
                    __syncwarp();
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (CTAS == 2) mbar_arrive_cluster(cluster_map(&tempty[acc], 0));
                else mbar_arrive(&tempty[acc]);
            }
            acc ^= 1;
            if (acc == 0) acc_ph ^= 1u;
        }
        // The CTA may exit once its stores have read their shared memory.
        if (lane == 0) bulk_wait_group_read<0>();
        __syncwarp();
    }
    tc_fence_before();
    __syncwarp();
    // A pair: both CTAs are done with TMEM and with each other's barriers.
    if constexpr (CTAS == 2) cluster_sync_all();
    else __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        if constexpr (CTAS == 2) tmem_dealloc_pair(tmem_base, 2 * kAccStride);
        else tmem_dealloc(tmem_base, 2 * kAccStride);
    }
}

template <int CTAS, int BN, int GROUPS>
void run_tile(const RoutedProduct& p, int min_rows, DeviceState& state, cudaStream_t stream) {
    using L = TileSmem<CTAS, BN, GROUPS>;
    TileMaps maps;
    const auto f16 = CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const auto sw = CU_TENSOR_MAP_SWIZZLE_128B;
    encode_tensor_map_2d(&maps.x, f16, p.x, p.k, p.x_rows, p.ldx * 2, BK, BM, sw);
    encode_tensor_map_2d(&maps.w, f16, p.operand, p.k, static_cast<uint64_t>(p.groups) * p.n,
                         static_cast<uint64_t>(p.k) * 2, BK, BN / CTAS, sw);
    if (p.y_type == SAMQ_TYPE_F16)
        encode_tensor_map_2d(&maps.y, f16, p.y, p.n, p.rows, p.ldy * 2, 64, 32, sw);
    else
        encode_tensor_map_2d(&maps.y, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, p.y, p.n, p.rows, p.ldy * 4, 32, 32, sw);
    maps.h = maps.x;
    maps.b = maps.w;
    if (p.ids) {
        encode_tensor_map_2d(&maps.h, f16, p.h2, 2 * p.rank, p.rows, 4 * p.rank, BK, BM, sw);
        encode_tensor_map_2d(&maps.b, f16, p.b2, 2 * p.rank, static_cast<uint64_t>(p.adapter_count) * p.n, 4 * p.rank,
                             BK, BN / CTAS, sw);
    }
    auto kernel = routed_tile_kernel<CTAS, BN, GROUPS>;
    const void* fn = reinterpret_cast<const void*>(kernel);
    set_smem_limit_once(state, fn, L::total, "cudaFuncSetAttribute(routed tile smem)");
    const int64_t tiles = (p.rows / (CTAS * BM) + p.groups) * ((p.n + BN - 1) / BN);  // at most
    if constexpr (CTAS == 2) {
        const int resident =
            pair_clusters_resident(state, fn, kThreads, L::total, "cudaOccupancyMaxActiveClusters(routed tile)");
        const int64_t pairs = std::min<int64_t>(tiles, resident);
        launch_pdl_pairs(kernel, dim3(static_cast<unsigned>(2 * pairs)), dim3(kThreads), L::total, stream,
                         "routed_tile_kernel launch", maps, p, min_rows, state.status);
    } else {
        const int64_t ctas = std::min<int64_t>(tiles, state.sm_count);
        launch_pdl(kernel, dim3(static_cast<unsigned>(ctas)), dim3(kThreads), L::total, stream,
                   "routed_tile_kernel launch", maps, p, min_rows, state.status);
    }
}

// A step of 64 columns takes a CTA pair on 256 x 256 and two single CTAs on 128 x
// 128 each the same time, as both shapes ask L2 for 32 KB an SM and step: the shape
// of fewer waves wins, and of equal ones the single CTA, which starts and ends
// sooner.  Row tiles: half a tile is lost at the end of every group.  Measured, waves
// pair : single, us pair : single: 1280 rows of 8 groups to n = 4096 2 : 4, 24.8 :
// 30.8; to n = 1024 1 : 1, 15.6 : 13.1; 2400 to n = 1024 1 : 2, 13.3 : 16.0; one group
// of 2000 to n = 1024 1 : 1, 12.6 : 10.3.  (256-wide single CTAs and pairs 128 or 192
// wide were nowhere more than 3% better.)
template <int GROUPS>
void run_shape(const RoutedProduct& p, int min_rows, DeviceState& state, cudaStream_t stream) {
    auto waves = [&](int64_t height, int64_t width, int64_t units) {
        const int64_t rows = p.groups > 1 ? p.rows + p.groups * height / 2 : p.rows + height - 1;
        const int64_t tiles = rows / height * ((p.n + width - 1) / width);
        return (tiles + units - 1) / units;
    };
    if (waves(2 * BM, 256, state.sm_count / 2) < waves(BM, 128, state.sm_count))
        run_tile<2, 256, GROUPS>(p, min_rows, state, stream);
    else
        run_tile<1, 128, GROUPS>(p, min_rows, state, stream);
}

}  // namespace

void launch_routed_tile(const RoutedProduct& p, int min_rows, DeviceState& state, cudaStream_t stream) {
    if (p.groups <= 128) run_shape<128>(p, min_rows, state, stream);
    else run_shape<1024>(p, min_rows, state, stream);
}

}  // namespace samq
