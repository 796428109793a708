// routed_rows.cu -- the routed product for groups of few rows (decoding): the
// packed weights of the groups in use stream through once and are decoded on the
// way, so HBM carries 0.56-1.06 bytes a weight instead of the 2 of the f16
// expansion the tiles of routed_tile.cu read.
//
// y[i] = act(W_g x[i] + bias_g + delta_i) with the factors swapped: a unit is one
// packet row tile (128 rows of the stacked weights) of one group by up to TOK of
// the group's rows, D[128][TOK] = W_tile . X^T in TMEM (tcgen05.mma M = 128,
// N = TOK), and for every adapter a that one of the rows names
// D += [B_a | B_a]_tile . [hi(H) | lo(H)]_a^T with zeros for the rows of others, as
// in routed_tile.cu.  What bounds it at full size is the packet stream; what bounds it at
// a few rows is the chain of one unit, so a cluster of SPLIT CTAs shares a unit's
// depth and adds its partial sums over distributed shared memory, in rank order:
// one launch, no atomics, no workspace.
//
// One CTA per SM, persistent over the units of all groups:
//   warp 0       packets, several contiguous ones by one bulk copy, then 128 x 64 of
//                B | B by TMA for each adapter step;
//   last warp    the same columns of X by TMA (rows by index through the row gather),
//                hi | lo of the adapter's rows by the row gather;
//   warp 1       TMEM owner; one thread issues the MMAs;
//   warps 2-5    epilogue: one weight row a lane, TMEM to registers (SPLIT > 1: to
//                shared memory of the CTA that adds up the row), bias, erf-GELU,
//                stores coalesced over the weight rows;
//   warps 6-     decoders, sets of four on steps of several packets in turn: a thread
//                turns a row of its packets into f16 with the values of packets.cuh bit
//                for bit and stores it to tensor memory, where the MMA takes it as its
//                left factor.
// Each copy and each step costs the one thread that issues it a round of waiting
// beside the decoders' many warps: hence several packets a copy and a step (the case
// below: 34.5 us with four, 36.8 with two, 43.6 with one), and one thread per kind of
// copy.
// The decoders' arithmetic spares the logic pipe, which runs at half rate: codes
// two at a time become halves by or-ing them into the mantissa of 1024 where they
// stand; the sum of such a half and -1024 as a float is exact and one operation of
// the full-rate pipe (add.f32.f16), and pairs of weights share packed f32 operations.
// An int8 is offset to be positive first, and f16(q d) needs a single half
// multiplication as q d has at most 19 bits.
// Measured (128 rows of 32 experts, 1024 -> 4096 Q4_K, two experts a row, GELU): 29 us
// for 75 MB of packets, 2.6 TB/s, 34.4 us with the rows' copy.  From a cold cache 38 us
// with the issue slots 52% busy (4.9 instructions a weight with the epilogue), the
// logic pipe 41% and the HBM 28%: no unit is full.  A quarter of the warps an SM could
// hold is there, and the rest of the time they wait on one another's hand-overs: the
// decoders bound it by latency, not the packet stream.
// A decoder set takes every kSets-th packet copy of a ring that carries the adapters'
// copies too, so it has not seen the earlier phases of the barrier it waits on, and
// a phase's parity alone cannot tell it from the one two before.  The packet
// producer has: it counts a copy as announced once it has found the stage free of
// the one before, and a set waits on a stage's barrier only after its own copy's
// announcement (a word of shared memory, read once for every few copies).  The
// barrier is then in that copy's phase, and cannot leave it before the set has
// decoded it.  (Waiting through every phase instead would not do: the phases of the
// other sets' copies may be gone by two when a set comes to them.)
// Every wait is bounded.  No load uses multicast.
#include <algorithm>
#include <climits>
#include <map>
#include <tuple>

#include "packets.cuh"
#include "samq_internal.hpp"

namespace samq {
namespace {

constexpr int kDecodeWarps = 12;
constexpr int kXWarp = 6 + kDecodeWarps;
constexpr int kThreads = 32 * (kXWarp + 1);
constexpr int kSets = kDecodeWarps / 4;
constexpr int kMaxGroups = 1024;
constexpr int kSmemLimit = 232448;
constexpr int kMaxSplit = 8;
constexpr int kMaxChunks = kRoutedFewAdapted / 64;  // row chunks of a call with adapters

template <int TYPE, int TOK>
struct RowsSmem {
    static constexpr int packet = 128 * (code_bytes_of(TYPE) + 8);
    static constexpr int depth = TOK == 64 ? 2 : 4;  // packets (64 columns each) of a copy and of a step
    static constexpr int slot = 32 * depth;          // TMEM columns of a step's left factor: 128 rows x 64 depth f16
    static constexpr int raw_bytes = depth * packet;
    static constexpr int b_bytes = 128 * 128;  // an adapter step's B | B, where the packets lie
    static constexpr int raw_stage = (raw_bytes > b_bytes ? raw_bytes : b_bytes + 1023) / 1024 * 1024;
    static constexpr int x_chunk = TOK * 128;  // 64 columns of TOK rows
    static constexpr int x_bytes = depth * x_chunk;
    static constexpr int part = TOK * 128 * 4;  // partial sums [TOK][128]
    static constexpr int tables = (3 * kMaxGroups + 1) * 4;
    static constexpr int lists = kMaxChunks * (TOK + 1) * 4;  // the adapters of each row chunk and how many
    static constexpr int fixed = 1024 + part + 512 + tables + lists;
    static constexpr int fit = (kSmemLimit - fixed) / (raw_stage + x_bytes);
    static constexpr int stages = fit > 8 ? 8 : fit;
    static constexpr int slots = (512 - 2 * TOK) / slot;  // left factors
    static constexpr int raw_off = stages * x_bytes;
    static constexpr int part_off = raw_off + stages * raw_stage;
    static constexpr int bar_off = part_off + part;
    static constexpr int table_off = bar_off + 512;
    static constexpr int list_off = table_off + tables;
    static constexpr int total = fixed + stages * (raw_stage + x_bytes);
};

__device__ __forceinline__ uint32_t half2_of(uint64_t v) {
    float a, b;
    unpack2(v, a, b);
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// Two halves with the bits of `mask` in their mantissas: one three-input logic
// operation.  `magic` is 1024 twice, in a register: as a second constant beside the
// mask it would make two operations.
__device__ __forceinline__ uint32_t or_into(uint32_t v, uint32_t mask, uint32_t magic) { return (v & mask) | magic; }
// The lower and the upper half of v, plus c, as floats.
__device__ __forceinline__ float low_plus(uint32_t v, float c) {
    float d;
    asm("add.rn.f32.f16 %0, %1, %2;" : "=f"(d) : "h"(static_cast<uint16_t>(v)), "f"(c));
    return d;
}
__device__ __forceinline__ float high_plus(uint32_t v, float c) {
    float d;
    asm("add.rn.f32.f16 %0, %1, %2;" : "=f"(d) : "h"(static_cast<uint16_t>(v >> 16)), "f"(c));
    return d;
}
// v + f (h - 1024) in halves (whole numbers below 2048 here: exact).
__device__ __forceinline__ uint32_t add_field(uint32_t v, uint32_t h, float f) {
    const __half2 low = __hadd2(*reinterpret_cast<const __half2*>(&h), __floats2half2_rn(-1024.0f, -1024.0f));
    const __half2 sum = __hfma2(low, __floats2half2_rn(f, f), *reinterpret_cast<const __half2*>(&v));
    return *reinterpret_cast<const uint32_t*>(&sum);
}

// A packet row (codes `code`, scale record `rec`) as f16: word i of `out` holds
// columns 2 i and 2 i + 1 of the 64.
template <int TYPE>
__device__ __forceinline__ void decode_row(const uint8_t* __restrict__ code, const uint8_t* __restrict__ rec,
                                           uint32_t magic, uint32_t (&out)[32]) {
    const uint2 record = *reinterpret_cast<const uint2*>(rec);
    if constexpr (TYPE == SAMQ_TYPE_Q8_0) {
        const __half2 bias = __floats2half2_rn(-1152.0f, -1152.0f);  // 1024 of the mantissa trick, 128 of the sign
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<uint4*>(w + 4 * i) = *reinterpret_cast<const uint4*>(code + 16 * i);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const __half2 d = __half2half2(__ushort_as_half(static_cast<uint16_t>(i < 8 ? record.x : record.x >> 16)));
            const uint32_t u = w[i] ^ 0x80808080u;
            const uint32_t lo = __byte_perm(u, 0x64646464u, 0x4140), hi = __byte_perm(u, 0x64646464u, 0x4342);
            const __half2 a = __hmul2(__hadd2(*reinterpret_cast<const __half2*>(&lo), bias), d);
            const __half2 b = __hmul2(__hadd2(*reinterpret_cast<const __half2*>(&hi), bias), d);
            out[2 * i] = *reinterpret_cast<const uint32_t*>(&a);
            out[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&b);
        }
    } else {
        // Words of 8 nibbles (column 8 j + i at bit 4 i).
        uint32_t lo[8];
        if constexpr (TYPE == SAMQ_TYPE_Q5_K) {  // 40-byte rows
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<uint2*>(lo + 2 * i) = *reinterpret_cast<const uint2*>(code + 8 * i);
        } else {
            *reinterpret_cast<uint4*>(lo) = *reinterpret_cast<const uint4*>(code);
            *reinterpret_cast<uint4*>(lo + 4) = *reinterpret_cast<const uint4*>(code + 16);
        }
        uint32_t high[4] = {};
        if constexpr (TYPE == SAMQ_TYPE_Q6_K)  // 2 bits a column
            *reinterpret_cast<uint4*>(high) = *reinterpret_cast<const uint4*>(code + 32);
        if constexpr (TYPE == SAMQ_TYPE_Q5_K)  // 1 bit a column
            *reinterpret_cast<uint2*>(high) = *reinterpret_cast<const uint2*>(code + 32);
        const float d = __half2float(__ushort_as_half(static_cast<uint16_t>(record.x)));
        const float dmin = __half2float(__ushort_as_half(static_cast<uint16_t>(record.x >> 16)));
        float ds = 0.0f;
        uint64_t scale = 0, m2 = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            // The sub-block's scale, and a sixteenth of it for odd columns, which stand 4 bits further up.
            if (TYPE == SAMQ_TYPE_Q6_K ? j % 2 == 0 : j % 4 == 0) {
                if constexpr (TYPE == SAMQ_TYPE_Q6_K) {
                    const uint32_t sc = j < 4 ? record.x >> (16 + 8 * (j >> 1)) : record.y >> (8 * ((j >> 1) - 2));
                    ds = __fmul_rn(d, static_cast<float>(static_cast<int8_t>(sc & 0xffu)));
                } else {
                    const int h = j >> 2;
                    ds = __fmul_rn(d, static_cast<float>((record.y >> (8 * h)) & 0xffu));
                    const float dm = __fmul_rn(dmin, static_cast<float>((record.y >> (16 + 8 * h)) & 0xffu));
                    m2 = pack2(-dm, -dm);
                }
                scale = pack2(ds, ds * 0.0625f);
            }
            // v[i]: columns i and i + 4 in its halves, times 16 for odd i.
            const uint32_t n = lo[j];
            uint32_t v[4];
            v[0] = or_into(n, 0x000f000fu, magic);
            v[1] = or_into(n, 0x00f000f0u, magic);
            v[2] = or_into(n >> 8, 0x000f000fu, magic);
            v[3] = or_into(n >> 8, 0x00f000f0u, magic);
            if constexpr (TYPE == SAMQ_TYPE_Q5_K) {
                // Bits 0-3 of the byte to bits 0-3, bits 4-7 to bits 16-19.
                const uint32_t byte = (high[j >> 2] >> (8 * (j & 3))) & 0xffu, b = byte | (byte << 12);
                v[0] = add_field(v[0], or_into(b, 0x00010001u, magic), 16.0f);
                v[1] = add_field(v[1], or_into(b, 0x00020002u, magic), 128.0f);
                v[2] = add_field(v[2], or_into(b, 0x00040004u, magic), 4.0f);
                v[3] = add_field(v[3], or_into(b, 0x00080008u, magic), 32.0f);
            }
            if constexpr (TYPE == SAMQ_TYPE_Q6_K) {
                // The byte of columns 0-3 to bits 0-7, that of 4-7 to bits 16-23.
                const uint32_t b = __byte_perm(high[j >> 1], 0, j & 1 ? 0x4342 : 0x4140);
                v[0] = add_field(v[0], or_into(b, 0x00030003u, magic), 16.0f);
                v[1] = add_field(v[1], or_into(b, 0x000c000cu, magic), 64.0f);
                v[2] = add_field(v[2], or_into(b, 0x00300030u, magic), 1.0f);
                v[3] = add_field(v[3], or_into(b, 0x00c000c0u, magic), 4.0f);
            }
            constexpr float even = TYPE == SAMQ_TYPE_Q6_K ? -1024.0f - 32.0f : -1024.0f;
            constexpr float odd = TYPE == SAMQ_TYPE_Q6_K ? -1024.0f - 512.0f : -1024.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t ve = v[2 * (i & 1)], vo = v[2 * (i & 1) + 1];
                const uint64_t q = i < 2 ? pack2(low_plus(ve, even), low_plus(vo, odd))
                                         : pack2(high_plus(ve, even), high_plus(vo, odd));
                // ds q has at most 22 bits, so the fused form rounds where the separate one does
                if constexpr (TYPE == SAMQ_TYPE_Q6_K) out[4 * j + i] = half2_of(mul2(q, scale));
                else out[4 * j + i] = half2_of(fma2(q, scale, m2));
            }
        }
    }
}

__device__ __forceinline__ void gather4(void* dst, const CUtensorMap* map, uint64_t* bar, int x, const int (&r)[4]) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, "
        "%5, %6, %7}], [%2];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3])
        : "memory");
}

// A shared::cta address as that of CTA `rank` of the cluster, and a store there.
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, int rank) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
    return remote;
}
__device__ __forceinline__ void st_cluster(uint32_t addr, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

// Copies announced by the packet producer (a count in this CTA's shared memory).
__device__ __forceinline__ void announce(int* count, int copies) {
    asm volatile("st.release.cta.shared::cta.u32 [%0], %1;" ::"r"(smem_u32(count)), "r"(copies) : "memory");
}
__device__ __forceinline__ int announced(const int* count) {
    int copies;
    asm volatile("ld.acquire.cta.shared::cta.u32 %0, [%1];" : "=r"(copies) : "r"(smem_u32(count)) : "memory");
    return copies;
}
// Bounded wait until more than `copy` copies are announced, returning their number;
// at most `copy` when the wait is abandoned.
__device__ __forceinline__ int wait_announced(const int* count, int copy, DeviceStatus* status, uint32_t site) {
    int copies = announced(count);
    if (copies > copy) return copies;
    const uint64_t start = global_timer_ns();
    for (uint32_t spin = 1;; ++spin) {
        copies = announced(count);
        if (copies > copy) return copies;
        __nanosleep(32);
        if ((spin & 15u) == 0 && global_timer_ns() - start > kWaitTimeoutNs) {
            if (status) {
                atomicOr(&status->flags, kStatusTimeout);
                atomicExch(&status->timeout_site, site);
            }
            return copies;
        }
    }
}

__device__ __forceinline__ int clamp_row(int v, int64_t rows) {
    return v < 0 ? 0 : v > rows ? static_cast<int>(rows) : v;
}

// Packet row tiles that hold rows of group g.
__device__ __forceinline__ int first_tile(int g, int n) { return static_cast<int>(static_cast<int64_t>(g) * n / 128); }
__device__ __forceinline__ int group_tiles(int g, int n) {
    return static_cast<int>((static_cast<int64_t>(g + 1) * n - 1) / 128) - first_tile(g, n) + 1;
}

struct Unit {
    int group, tile, row0, count;  // packet row tile of the stacked weights, plan rows row0 .. row0 + count - 1
    int chunk;                     // of the group's rows
};

// Warp-collective: the last group whose first unit is at most `unit`, by two
// ballots (every 32nd group, then the 32 behind it).
template <int TOK>
__device__ __forceinline__ Unit find_unit(int unit, int n, int groups, const int* s_first, const int* s_begin,
                                          const int* s_end, int lane) {
    int lo = 0;
    if (groups > 1) {
        if (groups > 32) {
            const bool below = 32 * lane < groups && s_first[32 * lane] <= unit;
            lo = 32 * (__popc(__ballot_sync(0xffffffffu, below)) - 1);
        }
        const bool below = lo + lane < groups && s_first[lo + lane] <= unit;
        lo += __popc(__ballot_sync(0xffffffffu, below)) - 1;
    }
    const int tiles = group_tiles(lo, n), at = unit - s_first[lo];
    Unit u;
    u.group = lo;
    u.chunk = at / tiles;
    u.tile = first_tile(lo, n) + at - u.chunk * tiles;
    u.row0 = s_begin[lo] + u.chunk * TOK;
    u.count = min(TOK, s_end[lo] - u.row0);
    return u;
}

template <int TYPE, int TOK>
__global__ void __launch_bounds__(kThreads, 1)
routed_rows_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_h,
                   const __grid_constant__ CUtensorMap map_b, const RoutedProduct p, int max_rows, int split,
                   DeviceStatus* status) {
    using L = RowsSmem<TYPE, TOK>;
    constexpr int kStages = L::stages, kSlots = L::slots, kDepth = L::depth, kTmemStep = L::slot;
    static_assert(kStages >= 2 && kSlots >= kSets && L::total <= kSmemLimit, "shared memory budget");
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sx = smem;
    uint8_t* sraw = smem + L::raw_off;
    float* spart = reinterpret_cast<float*>(smem + L::part_off);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::bar_off);
    uint64_t* empty = full + kStages;
    uint64_t* a_full = empty + kStages;
    uint64_t* a_empty = a_full + kSlots;
    uint64_t* tfull = a_empty + kSlots;
    uint64_t* tempty = tfull + 2;
    uint64_t* part_full = tempty + 2;     // every CTA of the cluster has sent its partial sums here
    uint64_t* part_free = part_full + 1;  // every CTA has added up what it was sent
    uint64_t* drain = part_free + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    int* s_announced = reinterpret_cast<int*>(tmem_slot + 1);
    static_assert((2 * kStages + 2 * kSlots + 4 + 3) * 8 + 8 <= 512, "barrier space");
    static_assert(kSlots % kSets == 0, "a set follows every phase of the slots it fills");
    int* s_begin = reinterpret_cast<int*>(smem + L::table_off);
    int* s_end = s_begin + kMaxGroups;
    int* s_first = s_end + kMaxGroups;
    int* s_count = reinterpret_cast<int*>(smem + L::list_off);  // adapters of each row chunk
    int* s_list = s_count + kMaxChunks;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = split > 1 ? static_cast<int>(cluster_cta_rank()) : 0;
    const int cluster = blockIdx.x / split, clusters = gridDim.x / split;
    const int chunks = (p.k + 63) / 64;
    const int all_steps = (chunks + kDepth - 1) / kDepth;
    const int per = (all_steps + split - 1) / split;  // steps of a rank (the host leaves none without)
    const int step0 = rank * per, steps = min(all_steps, step0 + per) - step0;
    constexpr uint32_t kTmemCols = 512;  // 2 x TOK accumulator columns, then the left factors
    constexpr uint32_t kTmemA = 2 * TOK;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&full[s], 2);
            mbar_init(&empty[s], 1);
        }
        for (int s = 0; s < kSlots; ++s) {
            mbar_init(&a_full[s], 4);
            mbar_init(&a_empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&tfull[b], 1);
            mbar_init(&tempty[b], 4);
        }
        mbar_init(part_full, 4 * split);
        mbar_init(part_free, 4 * split);
        mbar_init(drain, 1);
        *s_announced = kStages;  // the first copies find their stages free
        fence_barrier_init();
        tma_prefetch_desc(&map_x);
    }
    if (warp == 1) tmem_alloc(tmem_slot, kTmemCols);
    // What the previous kernel may write is read from here on.  With adapters that
    // kernel is the down product, which began its own work only after everything
    // before it had completed: all but its pairs may be read at once, and the X
    // producer waits for those.
    if (!p.ids) pdl_wait();
    if (warp == 2) {
        int carry = 0;
        for (int base = 0; base < p.groups; base += 32) {
            const int g = base + lane;
            int begin = 0, end = 0, units = 0;
            if (g < p.groups) {
                begin = p.offsets ? clamp_row(__ldg(p.offsets + g), p.rows) : 0;
                end = p.offsets ? max(begin, clamp_row(__ldg(p.offsets + g + 1), p.rows)) : static_cast<int>(p.rows);
                units = end - begin <= max_rows ? (end - begin + TOK - 1) / TOK * group_tiles(g, p.n) : 0;
                s_begin[g] = begin;
                s_end[g] = end;
            }
            int sum = units;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += u;
            }
            if (g < p.groups) s_first[g] = carry + sum - units;
            carry += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (lane == 0) s_first[p.groups] = carry;
    }
    if (p.ids && warp >= 6 && warp - 6 < kMaxChunks) {
        // The adapters of row chunk `warp - 6`, in rising order.
        const int chunk = warp - 6, row0 = chunk * TOK;
        int id[(TOK + 31) / 32], found = 0, last = -1;
#pragma unroll
        for (int j = 0; j < (TOK + 31) / 32; ++j) {
            const int t = 32 * j + lane;
            id[j] = t < TOK && row0 + t < p.rows ? __ldg(p.ids + row0 + t) : -1;
        }
        for (;;) {
            int next = p.adapter_count;
#pragma unroll
            for (int j = 0; j < (TOK + 31) / 32; ++j)
                if (id[j] > last) next = min(next, id[j]);
            next = __reduce_min_sync(0xffffffffu, next);
            if (next >= p.adapter_count) break;
            if (lane == 0) s_list[chunk * TOK + found] = next;
            ++found;
            last = next;
        }
        if (lane == 0) s_count[chunk] = found;
    }
    tc_fence_before();
    if (split > 1) cluster_sync_all();
    else __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int units = s_first[p.groups];
    // A unit's steps of this rank: `steps` of packets, then adapter steps rank, rank + split, ... of the
    // chunk's adapters x the 64-column pieces of their pair.
    const int pieces = p.ids ? (2 * p.rank + 63) / 64 : 0;
    auto adapter_steps = [&](int chunk) {
        const int all = p.ids ? s_count[chunk] * pieces : 0;
        return all > rank ? (all - rank + split - 1) / split : 0;
    };

    if (warp == 0 || warp == kXWarp) {
        const bool is_x = warp == kXWarp;
        int before = 0;  // copies before this unit: copy i uses stage (before + i) % kStages
        bool ok = true;
        for (int unit = cluster; unit < units && ok; unit += clusters) {
            const Unit u = find_unit<TOK>(unit, p.n, p.groups, s_first, s_begin, s_end, lane);
            const int more = adapter_steps(u.chunk);
            int s = before % kStages;
            uint32_t ph = static_cast<uint32_t>(before / kStages) & 1u;
            auto advance = [&] {
                if (++s == kStages) {
                    s = 0;
                    ph ^= 1u;
                }
            };
            if (!is_x) {
                // One thread issues the unit's packets and adapter tiles.
                if (elect_one()) {
                    const int left = min(chunks - step0 * kDepth, steps * kDepth);
                    const uint8_t* from =
                        p.packets + (static_cast<int64_t>(u.tile) * chunks + step0 * kDepth) * L::packet;
                    for (int c = 0, copy = before; c < left; c += kDepth) {
                        if (!(ok = mbar_wait(&empty[s], ph ^ 1u, status, 71))) break;
                        if (++copy > kStages) announce(s_announced, copy);
                        const int bytes = min(kDepth, left - c) * L::packet;
                        mbar_arrive_expect_tx(&full[s], bytes);
                        bulk_load_1d(sraw + s * L::raw_stage, from, bytes, &full[s]);
                        from += L::raw_bytes;
                        advance();
                    }
                    for (int i = 0; i < more && ok; ++i) {
                        if (!(ok = mbar_wait(&empty[s], ph ^ 1u, status, 71))) break;
                        const int at = rank + i * split;
                        const int a = s_list[u.chunk * TOK + at / pieces];
                        mbar_arrive_expect_tx(&full[s], L::b_bytes);
                        tma_load_2d(sraw + s * L::raw_stage, &map_b, &full[s], at % pieces * 64,
                                    a * p.n + u.tile * 128);
                        advance();
                    }
                }
                __syncwarp();
            } else {
                if (!p.row_index) {
                    if (elect_one())
                        for (int c = step0 * kDepth; c < min(chunks, (step0 + steps) * kDepth); c += kDepth) {
                            if (!(ok = mbar_wait(&empty[s], ph ^ 1u, status, 71))) break;
                            if (p.k % 64 == 0) {  // one copy; the chunks past the end read zeros
                                mbar_arrive_expect_tx(&full[s], L::x_bytes);
                                tma_load_3d(sx + s * L::x_bytes, &map_x, &full[s], 0, u.row0, c);
                            } else {
                                const int here = min(kDepth, chunks - c);
                                mbar_arrive_expect_tx(&full[s], here * L::x_chunk);
                                for (int j = 0; j < here; ++j)
                                    tma_load_2d(sx + s * L::x_bytes + j * L::x_chunk, &map_x, &full[s], (c + j) * 64,
                                                u.row0);
                            }
                            advance();
                        }
                    __syncwarp();
                }
                // Rows by index and adapter rows: four rows a lane.
                const int first = p.row_index ? 0 : steps;
                ok = __all_sync(0xffffffffu, ok);
                if (ok && first < steps + more) {
                    int rows[4], id[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int at = u.row0 + 4 * lane + j;
                        const bool in = 4 * lane + j < u.count;
                        const int r = p.row_index && in ? __ldg(p.row_index + at) : -1;
                        rows[j] = r >= 0 && r < p.x_rows ? r : static_cast<int>(p.x_rows);  // past the end: zeros
                        id[j] = p.ids && in ? __ldg(p.ids + at) : -1;
                    }
                    if (more) pdl_wait();  // the pairs of the down product
                    s = (before + first) % kStages;
                    ph = static_cast<uint32_t>((before + first) / kStages) & 1u;
                    for (int i = first; i < steps + more; ++i) {
                        if (elect_one()) ok = mbar_wait(&empty[s], ph ^ 1u, status, 71);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        if (i < steps) {
                            const int c0 = (step0 + i) * kDepth, here = min(kDepth, chunks - c0);
                            if (elect_one()) mbar_arrive_expect_tx(&full[s], here * L::x_chunk);
                            __syncwarp();
                            if (lane < TOK / 4)
                                for (int c = 0; c < here; ++c)
                                    gather4(sx + s * L::x_bytes + c * L::x_chunk + lane * 512, &map_x, &full[s],
                                            (c0 + c) * 64, rows);
                        } else {
                            const int at = rank + (i - steps) * split;
                            const int a = s_list[u.chunk * TOK + at / pieces];
                            if (elect_one()) mbar_arrive_expect_tx(&full[s], L::x_chunk);
                            __syncwarp();
                            if (lane < TOK / 4) {
                                int from[4];
#pragma unroll
                                for (int j = 0; j < 4; ++j)
                                    from[j] = id[j] == a ? u.row0 + 4 * lane + j : static_cast<int>(p.rows);
                                gather4(sx + s * L::x_bytes + lane * 512, &map_h, &full[s], at % pieces * 64, from);
                            }
                        }
                        advance();
                    }
                }
            }
            ok = __all_sync(0xffffffffu, ok);
            before += steps + more;
        }
        if (is_x) pdl_wait();  // if not before: the kernel ends after its predecessors
        pdl_trigger();  // this warp's loads are issued
        if (!ok && lane == 0) {
            // A wait gave up: time for the copies in flight to land before the CTA exits.
            const uint64_t start = global_timer_ns();
            while (global_timer_ns() - start < 2000000ull) __nanosleep(1000);
        }
        __syncwarp();
    } else if (warp == 1) {
        if (elect_one()) {
            constexpr uint32_t idesc = idesc_f16_f32(128, TOK);
            const uint64_t x_desc = smem_desc_sw128(smem_u32(sx)), b_desc = smem_desc_sw128(smem_u32(sraw));
            int s = 0, slot = 0, acc = 0;
            uint32_t ph = 0, slot_ph = 0, acc_ph = 0;
            bool ok = true;
            auto advance = [&] {
                if (++s == kStages) {
                    s = 0;
                    ph ^= 1u;
                }
            };
            for (int unit = cluster; unit < units && ok; unit += clusters) {
                if (!mbar_wait(&tempty[acc], acc_ph ^ 1u, status, 72)) break;
                tc_fence_after();
                const uint32_t d = tmem_base + static_cast<uint32_t>(acc * TOK);
                for (int i = 0; i < steps; ++i) {
                    if (!mbar_wait(&full[s], ph, status, 73) || !mbar_wait(&a_full[slot], slot_ph, status, 74)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t a = tmem_base + kTmemA + static_cast<uint32_t>(slot * kTmemStep);
                    const uint64_t xd = x_desc + static_cast<uint32_t>(s * (L::x_bytes >> 4));
                    const int here = min(kDepth, chunks - (step0 + i) * kDepth);
#pragma unroll
                    for (int c = 0; c < kDepth; ++c)
                        if (c < here)
#pragma unroll
                            for (int kk = 0; kk < 4; ++kk)
                                tc_mma_f16_ts(d, a + 32 * c + 8 * kk, xd + c * (L::x_chunk >> 4) + 2 * kk, idesc,
                                              i | c | kk ? 1u : 0u);
                    tc_commit(&a_empty[slot]);
                    if (++slot == kSlots) {
                        slot = 0;
                        slot_ph ^= 1u;
                    }
                    tc_commit(&empty[s]);
                    advance();
                }
                const int more = ok && p.ids ? adapter_steps(unit / group_tiles(0, p.n)) : 0;
                for (int i = 0; i < more; ++i) {
                    if (!mbar_wait(&full[s], ph, status, 73)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint64_t bd = b_desc + static_cast<uint32_t>(s * (L::raw_stage >> 4));
                    const uint64_t xd = x_desc + static_cast<uint32_t>(s * (L::x_bytes >> 4));
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) tc_mma_f16(d, bd + 2 * kk, xd + 2 * kk, idesc, 1u);
                    tc_commit(&empty[s]);
                    advance();
                }
                if (!ok) break;
                tc_commit(&tfull[acc]);
                acc ^= 1;
                if (acc == 0) acc_ph ^= 1u;
            }
            tc_commit(drain);  // every MMA this thread issued is complete before TMEM is released
            mbar_wait(drain, 0, status, 76);
        }
        __syncwarp();
    } else if (warp >= 6) {
        // The CTA's packet steps go to the sets and slots in turn.
        const int set = (warp - 6) >> 2;
        const int quarter = warp & 3;  // the TMEM lanes a warp may store to
        const int r = quarter * 32 + lane;
        const uint32_t lanes = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + kTmemA;
        const uint32_t magic = 0x64006400u + threadIdx.z;  // the compiler does not know that threadIdx.z is 0
        int done = 0;    // packet steps before this unit
        int copies = 0;  // copies of either kind before this unit
        int known = kStages;  // copies known to be announced
        bool ok = true;
        for (int unit = cluster; unit < units && ok; unit += clusters) {
            int i = set - done % kSets;
            if (i < 0) i += kSets;  // this set's first step of the unit
            for (; i < steps; i += kSets) {
                const int copy = copies + i, s = copy % kStages;
                const int step = done + i, slot = step % kSlots;
                if (!mbar_wait(&a_empty[slot], (static_cast<uint32_t>(step / kSlots) & 1u) ^ 1u, status, 78)) ok = false;
                else if (copy >= known && (known = wait_announced(s_announced, copy, status, 75)) <= copy) ok = false;
                else ok = mbar_wait(&full[s], static_cast<uint32_t>(copy / kStages) & 1u, status, 77);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                const int here = min(kDepth, chunks - (step0 + i) * kDepth);
                for (int c = 0; c < here; ++c) {
                    const uint8_t* raw = sraw + s * L::raw_stage + c * L::packet;
                    uint32_t w[32];
                    decode_row<TYPE>(raw + r * code_bytes_of(TYPE), raw + 128 * code_bytes_of(TYPE) + r * 8, magic, w);
                    tc_st_32x32b_x32(lanes + static_cast<uint32_t>(slot * kTmemStep + 32 * c), w);
                }
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&a_full[slot]);
            }
            done += steps;
            copies += steps;
            if (p.ids) copies += adapter_steps(unit / group_tiles(0, p.n));  // one group
        }
    } else {
        const int quarter = warp & 3;  // TMEM lanes 32 * quarter ..
        const int mine = quarter * 32 + lane;
        const bool f16 = p.y_type == SAMQ_TYPE_F16;
        const int elem = f16 ? 2 : 4;
        const int64_t stride = p.ldy * elem;
        const int shift = 31 - __clz(split);  // split is a power of two
        const int share = TOK >> shift;       // rows that a CTA of the cluster finishes: t % split == rank
        int acc = 0;
        uint32_t acc_ph = 0, part_ph = 0;
        // The next unit's place and bias are fetched under this one's wait.
        Unit u{}, next{};
        float bias = 0.0f, next_bias = 0.0f;
        auto fetch = [&](int unit) {
            if (unit >= units) return;
            next = find_unit<TOK>(unit, p.n, p.groups, s_first, s_begin, s_end, lane);
            const int64_t col = static_cast<int64_t>(next.tile) * 128 + mine - static_cast<int64_t>(next.group) * p.n;
            next_bias = p.bias && col >= 0 && col < p.n ? __ldg(p.bias + static_cast<int64_t>(next.group) * p.n + col)
                                                        : 0.0f;
        };
        fetch(cluster);
        for (int unit = cluster; unit < units; unit += clusters) {
            u = next;
            bias = next_bias;
            fetch(unit + clusters);
            // This lane's weight row as a column of the group's output.
            const int64_t col = static_cast<int64_t>(u.tile) * 128 + mine - static_cast<int64_t>(u.group) * p.n;
            const bool in = col >= 0 && col < p.n;
            uint8_t* out = static_cast<uint8_t*>(p.y) + (u.row0 * p.ldy + col) * elem;
            // Rows t and t + step (where `both`): their sums a and b through the epilogue and out.
            auto finish = [&](int t, int step, bool both, float a, float b) {
                a += bias;
                b += bias;
                if (p.gelu) gelu_erf2(a, b);
                uint8_t* at = out + t * stride;
                if (!in) return;
                if (f16) *reinterpret_cast<__half*>(at) = __float2half_rn(a);
                else *reinterpret_cast<float*>(at) = a;
                if (!both) return;
                at += step * stride;
                if (f16) *reinterpret_cast<__half*>(at) = __float2half_rn(b);
                else *reinterpret_cast<float*>(at) = b;
            };
            // Warp-uniform: the TMEM loads below are warp-collective.
            if (!__all_sync(0xffffffffu, mbar_wait(&tfull[acc], acc_ph, status, 79))) break;
            tc_fence_after();
            const uint32_t d = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(acc * TOK);
            constexpr int C = TOK < 32 ? TOK : 32;
            if (split > 1 &&
                !__all_sync(0xffffffffu, mbar_wait_cluster(part_free, part_ph ^ 1u, status, 80)))
                break;
#pragma unroll 1
            for (int c = 0; c < u.count; c += C) {
                uint32_t v[C];
                if constexpr (C == 16) tc_ld_32x32b_x16(d + c, v);
                else tc_ld_32x32b_x32(d + c, v);
                tc_wait_ld();
                if (split > 1) {
                    // Row t to CTA t % split: slot [this rank][t / split] of its partial sums.
                    const uint32_t slot = smem_u32(spart + rank * share * 128 + mine);
#pragma unroll
                    for (int i = 0; i < C; ++i) {
                        const int t = c + i;
                        if (t < u.count)
                            st_cluster(map_rank(slot + (t >> shift) * 512, t & (split - 1)), __uint_as_float(v[i]));
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < C; i += 2) {
                        if (c + i >= u.count) break;
                        finish(c + i, 1, c + i + 1 < u.count, __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
                    }
                }
                __syncwarp();  // converged for the next collective load
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&tempty[acc]);
            acc ^= 1;
            if (acc == 0) acc_ph ^= 1u;
            if (split > 1) {
                if (lane < split) mbar_arrive_cluster(cluster_map(part_full, lane));
                if (!__all_sync(0xffffffffu, mbar_wait_cluster(part_full, part_ph, status, 81))) break;
                for (int t = rank; t < u.count; t += 2 * split) {
                    const bool both = t + split < u.count;
                    const float* from = spart + (t >> shift) * 128 + mine;
                    float v0 = 0.0f, v1 = 0.0f;
                    for (int o = 0; o < split; ++o) {
                        v0 += from[o * share * 128];
                        if (both) v1 += from[o * share * 128 + 128];
                    }
                    finish(t, split, both, v0, v1);
                }
                __syncwarp();
                if (lane < split) mbar_arrive_cluster(cluster_map(part_free, lane));
                part_ph ^= 1u;
            }
        }
        tc_fence_before();
    }
    __syncwarp();
    // A cluster: nobody reads this CTA's shared memory any more.
    if (split > 1) cluster_sync_all();
    else __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, kTmemCols);
    }
}

// How many clusters of `split` CTAs of `kernel` can be resident on the device;
// queried once per (kernel, device, split).
int resident_clusters(DeviceState& state, const void* kernel, int split, int smem) {
    static std::mutex mutex;
    static std::map<std::tuple<const void*, int, int>, int> cache;
    std::lock_guard<std::mutex> lock(mutex);
    int& clusters = cache[{kernel, state.device, split}];
    if (clusters > 0) return clusters;
    DeviceGuard guard(state.device);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(split);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(split);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    check_cuda(cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg), "cudaOccupancyMaxActiveClusters(routed rows)");
    if (clusters <= 0) fail(SAMQ_ERR_CUDA, "no cluster of the routed rows kernel fits on this device");
    return clusters;
}

template <int TYPE, int TOK>
void run_rows(const RoutedProduct& p, int max_rows, DeviceState& state, cudaStream_t stream) {
    using L = RowsSmem<TYPE, TOK>;
    CUtensorMap map;
    const auto f16 = CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    if (!p.row_index && p.k % 64 == 0)  // [k / 64][x_rows][64]: several 64-column chunks a copy
        encode_tensor_map_3d_box(&map, f16, p.x, 64, p.x_rows, p.k / 64, p.ldx * 2, 128, 64, TOK, L::depth,
                                 CU_TENSOR_MAP_SWIZZLE_128B);
    else
        encode_tensor_map_2d(&map, f16, p.x, p.k, p.x_rows, p.ldx * 2, 64, p.row_index ? 1 : TOK,
                             CU_TENSOR_MAP_SWIZZLE_128B);
    CUtensorMap map_h = map, map_b = map;
    if (p.ids) {
        encode_tensor_map_2d(&map_h, f16, p.h2, 2 * p.rank, p.rows, 4 * p.rank, 64, 1,
                             CU_TENSOR_MAP_SWIZZLE_128B);
        encode_tensor_map_2d(&map_b, f16, p.b2, 2 * p.rank,
                             static_cast<uint64_t>(p.adapter_count) * p.n, 4 * p.rank, 64, 128,
                             CU_TENSOR_MAP_SWIZZLE_128B);
    }
    auto kernel = routed_rows_kernel<TYPE, TOK>;
    set_smem_limit_once(state, reinterpret_cast<const void*>(kernel), L::total,
                        "cudaFuncSetAttribute(routed rows smem)");
    const int tiles = (p.n + 127) / 128 + (p.n % 128 ? 1 : 0);  // of a group, at most
    const int64_t units = std::min<int64_t>(p.rows, p.groups + p.rows / TOK) * tiles;  // at most
    const int steps = ((p.k + 63) / 64 + L::depth - 1) / L::depth;
    const void* fn = reinterpret_cast<const void*>(kernel);
    // Few units: the widest cluster that still has every unit resident.
    int split = 1;
    for (int wide = 2; wide <= kMaxSplit && steps >= wide; wide *= 2) {
        const bool all_work = (wide - 1) * ((steps + wide - 1) / wide) < steps;  // no rank without steps
        if (all_work && units <= resident_clusters(state, fn, wide, L::total)) split = wide;
    }
    const int64_t clusters = std::min<int64_t>(units, split > 1 ? resident_clusters(state, fn, split, L::total) : state.sm_count);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(clusters * split));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = L::total;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(split);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    check_cuda(cudaLaunchKernelEx(&cfg, kernel, map, map_h, map_b, p, max_rows, split, state.status), "routed_rows_kernel launch");
}

template <int TYPE>
void run_type(const RoutedProduct& p, int max_rows, DeviceState& state, cudaStream_t stream) {
    const int64_t mean = (p.rows + p.groups - 1) / p.groups;
    if (mean <= 16) run_rows<TYPE, 16>(p, max_rows, state, stream);
    else if (mean <= 32) run_rows<TYPE, 32>(p, max_rows, state, stream);
    else run_rows<TYPE, 64>(p, max_rows, state, stream);
}

}  // namespace

void launch_routed_rows(const RoutedProduct& p, int max_rows, DeviceState& state, cudaStream_t stream) {
    switch (p.type) {
        case SAMQ_TYPE_Q8_0: run_type<SAMQ_TYPE_Q8_0>(p, max_rows, state, stream); break;
        case SAMQ_TYPE_Q4_K: run_type<SAMQ_TYPE_Q4_K>(p, max_rows, state, stream); break;
        case SAMQ_TYPE_Q5_K: run_type<SAMQ_TYPE_Q5_K>(p, max_rows, state, stream); break;
        default: run_type<SAMQ_TYPE_Q6_K>(p, max_rows, state, stream); break;
    }
}

}  // namespace samq
