// FP8 GEMM whose operands carry one FP32 scale for every block of 128 (A: 1 x 128, B: 128 x 128):
//   D[m, n] = C[m, n] + sum over K blocks of  sfa[m, kb] sfb[n / 128, kb] * sum_{k in kb} A[m, k] B[n, k]
// for the dense, m-grouped (row ids or psum) and masked layouts. The tensor core's block-scaled kinds take power-of-two scales
// only, so the products of one K block are summed by tcgen05.mma (kind::f8f6f4) into an accumulator of their own in
// tensor memory, and the epilogue warps keep the running sum in registers: one FP32 multiply-add per element and K block with
// the product of the two scales. Behavioural counterpart in the reference: its FP32-scale kernel of the previous architecture
// (deep_gemm/include/deep_gemm/impls/sm90_fp8_gemm_1d2d.cuh), reached there with disable_ue8m0_cast.
//
// Warp roles (384 threads): warp 0 loads A tiles, warp 3 B tiles, warp 1 issues the MMAs, warp 2 owns the tensor memory and brings the scales,
// warps 4-11 add up (TMEM lane quarter = warp index % 4, two warps per quarter split the columns). A thread owns one row's
// half of the tile in registers, so a scale is one scalar per thread and K block and no value crosses lanes until the store.
//
// What bounds it: the sums. A K block of a 128 x 256 tile is 512 cycles of MMAs, and each scheduler has two warps that read 128 columns of
// tensor memory (60 cycles per 32 columns) and issue 64 packed multiply-adds (2.2 cycles each) for it, which take turns
// rather than overlap, plus what the hand-over costs. Measured on the way, 4096 x 4096 x 7168 on pairs: scales read by the summing warps
// 151 us; through a warp of their own, the MMA issuer's loop cut to one wait 124; fewer commits and counters 119; whole lines
// stored 116; the loop unrolled twice 111 (2170 TFLOP/s; 8192 x 7168 x 4096 216 us, 2230). The power-of-two kernel, whose
// scales the tensor core applies, takes 98: the power limit is then what stops it. Without the multiply-adds this one takes 97, with
// half of them 103. What did not help: 16 summing warps (contention for the same ports: 134), 32-column loads (registers spill), one lane
// polling for its warp (the divergence costs more), the halves of a tile on barriers of their own (no difference).
#pragma once

#include <cuda_bf16.h>

#include "gemm_kernel.cuh"
#include "ptx.cuh"

namespace dgb {

struct BlockScaledParams {
    const float* sfa;  // element (group, row, kb) at sfa[group * sfa_group_stride + row * sfa_row_stride + kb * sfa_k_stride]
    const float* sfb;  // element (group, nb, kb) likewise, nb = n / 128
    long long sfa_group_stride, sfa_row_stride, sfa_k_stride;
    long long sfb_group_stride, sfb_n_stride, sfb_k_stride;
    void* d;
    const float* c;  // FP32 output only: added to the product; may be d itself
    long long d_row_stride, c_row_stride;  // elements
    const int* layout;
    int mode;  // kModeDense / kModeRowIds / kModePsum / kModeMasked (A and D [G, m, *])
    int m, n, k, num_groups, alignment, store_padding;
    int b_mn_major;   // B is [groups, k, n] with n contiguous
    int sf_vec;       // a row's scales of four consecutive K blocks lie in 16 aligned bytes
    int a_box_rows;   // rows of A that one load brings: 128, or fewer where tiles have few (a tile takes as many loads as its rows need)
};

// kind::f8f6f4 descriptor: E4M3 operands (format 0), FP32 accumulator.
__host__ __device__ constexpr uint32_t make_idesc_e4m3_f32(uint32_t m, uint32_t n) {
    return (1u << 4) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

// Shared-memory descriptors of 128-byte-swizzled tiles whose 8-row groups are 1024 bytes apart, as two words: the upper one is the same
// for every tile, the lower one holds the address (and, MN-major, the 16 KB between 128-byte chunks along N).
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(uint32_t smem_addr, bool mn_major) {
    return ((smem_addr & 0x3ffffu) >> 4) | (mn_major ? (16384u >> 4) << 16 : 0u);
}

// D[tmem] = A B^T of one K block: four MMAs of K = 32, the first one overwrites D. kPair: on both CTAs of the pair.
template <bool kPair>
__device__ __forceinline__ void mma_k_block(uint32_t tmem_d, uint32_t a_lo, uint32_t b_lo, uint32_t b_step, uint32_t idesc) {
#pragma unroll
    for (uint32_t k4 = 0; k4 < 4; ++k4) {
        if constexpr (kPair)
            asm volatile(
                "{\n\t"
                ".reg .pred p;\n\t"
                ".reg .b64 a, b;\n\t"
                "mov.b64 a, {%1, %4};\n\t"
                "mov.b64 b, {%2, %4};\n\t"
                "setp.ne.b32 p, %5, 0;\n\t"
                "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], a, b, %3, p;\n\t"
                "}\n"
                :: "r"(tmem_d), "r"(a_lo + k4 * 2), "r"(b_lo + k4 * b_step), "r"(idesc), "n"(kDescHi), "r"(k4) : "memory");
        else
            asm volatile(
                "{\n\t"
                ".reg .pred p;\n\t"
                ".reg .b64 a, b;\n\t"
                "mov.b64 a, {%1, %4};\n\t"
                "mov.b64 b, {%2, %4};\n\t"
                "setp.ne.b32 p, %5, 0;\n\t"
                "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %3, p;\n\t"
                "}\n"
                :: "r"(tmem_d), "r"(a_lo + k4 * 2), "r"(b_lo + k4 * b_step), "r"(idesc), "n"(kDescHi), "r"(k4) : "memory");
    }
}

// Two FP32 multiply-adds in one instruction: each result is what fmaf gives.
__device__ __forceinline__ void fma_f32x2(float& a0, float& a1, uint32_t x0, uint32_t x1, float s) {
    asm volatile("{\n\t"
        ".reg .b64 x, s, a;\n\t"
        "mov.b64 x, {%2, %3};\n\t"
        "mov.b64 s, {%4, %4};\n\t"
        "mov.b64 a, {%0, %1};\n\t"
        "fma.rn.f32x2 a, x, s, a;\n\t"
        "mov.b64 {%0, %1}, a;\n\t"
        "}\n" : "+f"(a0), "+f"(a1) : "r"(x0), "r"(x1), "f"(s));
}

// Tiled 3-D loads (same rules as the 2-D ones): into this CTA's shared memory, completing on its own barrier or on one of the pair's.
__device__ __forceinline__ void tma_load_3d(void* smem_dst, const CUtensorMap* map, uint64_t* bar, int32_t x, int32_t y, int32_t z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        :: "r"(smem_u32(smem_dst)), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ void tma_load_3d_pair(void* smem_dst, const CUtensorMap* map, uint32_t bar_cluster_addr, int32_t x, int32_t y,
                                                 int32_t z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        :: "r"(smem_u32(smem_dst)), "l"(map), "r"(bar_cluster_addr), "r"(x), "r"(y), "r"(z) : "memory");
}

constexpr int kScaleKb = 4;  // K blocks whose scales are loaded together

// Scales of up to kScaleKb K blocks (`left` of them exist, 0 for the others): one 16-byte load where that is allowed. Lanes hold rows
// far apart, so that every load instruction costs 32 cache lookups whatever its width.
__device__ __forceinline__ void load_scales(const float* from, long long k_stride, int left, bool whole, float* to) {
    if (whole && left >= kScaleKb) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(from));
        to[0] = v.x, to[1] = v.y, to[2] = v.z, to[3] = v.w;
        return;
    }
#pragma unroll
    for (int i = 0; i < kScaleKb; ++i) to[i] = i < left ? __ldg(from + i * k_stride) : 0.0f;
}

template <int BLOCK_N, int kStages, bool kPair>
struct BlockScaledSmem {
    static constexpr int kSumWarps = 8;
    static constexpr int kAccums = BLOCK_N == 256 ? 2 : 4;  // accumulators in tensor memory: K blocks between the MMAs and the sums
    // A slot of scales is written for K block i when the MMAs of K block i - kAccums are complete, which had waited until every summing
    // warp had left K block i - 2 kAccums, the slot's last user.
    static constexpr int kScaleSlots = 2 * kAccums;
    static constexpr int kScaleSlotBytes = 2 * 128 * 4;  // [half of the tile's columns][row]
    static constexpr int kStagingBytes = 16 * 128;       // epilogue: 16 rows x 128 bytes of each summing warp
    static constexpr int kABytes = 128 * 128;
    static constexpr int kBBytes = BLOCK_N * 128 / (kPair ? 2 : 1);
    static constexpr int kOffA = 0;
    static constexpr int kOffB = kOffA + kStages * kABytes;
    static constexpr int kOffStage = kOffB + kStages * kBBytes;
    static constexpr int kOffScales = kOffStage + kSumWarps * kStagingBytes;
    static constexpr int kOffBar = kOffScales + kScaleSlots * kScaleSlotBytes;
    static constexpr int kNumBars = 2 * kStages + kAccums;
    static constexpr int kOffMisc = kOffBar + (kNumBars * 8 + 15) / 16 * 16;
    static constexpr int kOffGroups = kOffMisc + 16;
    static constexpr int kTotal = kOffGroups + 4 * kMaxCachedGroups * 4;
    static constexpr int kDynamicBytes = kTotal + 1024;  // slack to align the base to 1024 B
};

struct BlockScaledTile {
    int row0;   // first row of this CTA's 128 in the flattened A / D (masked: inside the group)
    int rows;   // rows of them to store; may be zero or negative for the second CTA of a pair
    int group;  // < 0: nothing to do, every role skips the tile
    int n0;
};

// Walks the output tiles. Groups come from the table that the prologue puts into shared memory: start row, rows to
// compute, running tile count and end of the rows with scales of each.
// `ctas`: CTAs that share a tile (a pair, or a cluster that splits the tile's K).
template <int BLOCK_N, bool kPair>
struct BlockScaledScheduler {
    static constexpr int kTileM = kPair ? 256 : 128;
    const BlockScaledParams& p;
    const int *start, *rows, *tiles_end;
    int num_n_blocks, tile, stride, sub, g;
    uint32_t n_magic;  // tile / num_n_blocks = its product's upper half, or one less: the summing warps ask for a tile between two others

    __device__ BlockScaledScheduler(const BlockScaledParams& params, const int* table, int ctas)
        : p(params), start(table), rows(table + kMaxCachedGroups), tiles_end(table + 2 * kMaxCachedGroups),
          num_n_blocks((params.n + BLOCK_N - 1) / BLOCK_N), tile(static_cast<int>(blockIdx.x) / ctas),
          stride(static_cast<int>(gridDim.x) / ctas), sub(kPair ? static_cast<int>(blockIdx.x & 1) * 128 : 0), g(0),
          n_magic(0xffffffffu / static_cast<uint32_t>((params.n + BLOCK_N - 1) / BLOCK_N)) {}

    __device__ __forceinline__ void split(int index, int& mb, int& nb) const {
        mb = static_cast<int>(__umulhi(static_cast<uint32_t>(index), n_magic));
        nb = index - mb * num_n_blocks;
        while (nb >= num_n_blocks) {
            nb -= num_n_blocks;
            ++mb;
        }
    }

    // Rows of a group from the layout words; whatever they hold, no row at or past p.m is named.
    // `scaled`: end of the rows that have scales, in front of the padding rows among the `count`.
    __device__ __forceinline__ static void group_extent(const BlockScaledParams& p, int group, int& first, int& count, int& scaled) {
        if (p.mode == kModeMasked) {
            first = 0;
            count = scaled = min(max(__ldg(p.layout + group), 0), p.m);
            return;
        }
        const int prev_end = group == 0 ? 0 : min(max(__ldg(p.layout + group - 1), 0), p.m);
        const int end = min(max(__ldg(p.layout + group), 0), p.m);
        const long long al = p.alignment;
        first = static_cast<int>(min((prev_end + al - 1) / al * al, static_cast<long long>(p.m)));
        const int last = p.store_padding ? static_cast<int>(min((end + al - 1) / al * al, static_cast<long long>(p.m))) : end;
        count = end > first ? last - first : 0;
        scaled = end;
    }

    __device__ bool next(BlockScaledTile& t) {
        if (p.mode == kModeDense || p.mode == kModeRowIds) {
            if (tile >= (p.m + kTileM - 1) / kTileM * num_n_blocks) return false;
            int mb, nb;
            split(tile, mb, nb);
            t.row0 = mb * kTileM + sub;
            t.rows = min(128, p.m - t.row0);
            t.n0 = nb * BLOCK_N;
            t.group = p.mode == kModeDense ? 0 : __ldg(p.layout + t.row0);  // (no pairs with row ids: t.row0 < p.m)
            if (t.group >= p.num_groups) {
                if (threadIdx.x == 0) report_error(kBadArgument, t.row0, t.group);
                t.group = -1;
            }
            tile += stride;
            return true;
        }
        g = group_of_tile(tiles_end, g, p.num_groups, tile);
        if (g >= p.num_groups) return false;
        int mb, nb;
        split(tile - (g == 0 ? 0 : tiles_end[g - 1]), mb, nb);
        t.row0 = start[g] + mb * kTileM + sub;
        t.rows = min(128, rows[g] - mb * kTileM - sub);
        t.n0 = nb * BLOCK_N;
        t.group = g;
        tile += stride;
        return true;
    }
};

// 128 x 72 + 256 x 216 = 384 x 168, what the block is launched with (the 256-wide forms spill one word)
constexpr int kRegsBsControl = 72, kRegsBsSum = 216;

// kSplitK (dense form): the CTAs of a cluster (2, 4 or 8) share one tile and take a part of its K blocks each; every CTA leaves its sums in its
// own shared memory (the operand ring is done with), then the cluster adds them up, rank by rank in a fixed order. For problems
// with so few tiles that most SMs would idle while a few pull all of B.
template <int BLOCK_N, int kStages, bool kF32, bool kPair, bool kSplitK = false>
__global__ void __launch_bounds__(kGemmThreads, 1)
dgb200_block_scaled_gemm_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                                const __grid_constant__ BlockScaledParams p) {
    using L = BlockScaledSmem<BLOCK_N, kStages, kPair>;
    using Sched = BlockScaledScheduler<BLOCK_N, kPair>;
    constexpr int kCtas = kPair ? 2 : 1;
    constexpr int kAccums = L::kAccums;
    constexpr uint32_t kAccumCols = BLOCK_N < 64 ? 64 : BLOCK_N;
    constexpr int kSumWarps = L::kSumWarps;
    constexpr int kThreads = kGemmThreads;
    constexpr int kCols = BLOCK_N / (kSumWarps / 4);  // columns a thread sums
    static_assert(BLOCK_N == 32 || BLOCK_N == 64 || BLOCK_N == 128 || BLOCK_N == 256, "tile width");
    static_assert(!kPair || BLOCK_N == 256, "pairs work on 256 x 256 tiles");
    static_assert(!kSplitK || (!kPair && kStages * (L::kABytes + L::kBBytes) >= 128 * BLOCK_N * 4), "the operand ring holds the FP32 tile");
    static_assert(L::kDynamicBytes <= 232448, "shared memory budget");

    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + L::kOffBar);
    uint64_t* empty_bar = full_bar + kStages;
    uint64_t* tmem_full_bar = empty_bar + kStages;
    uint32_t* tmem_ptr_smem = reinterpret_cast<uint32_t*>(smem + L::kOffMisc);
    volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(smem + L::kOffMisc + 4);
    int* table = reinterpret_cast<int*>(smem + L::kOffGroups);

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t cta_rank = kPair ? cluster_cta_rank() : 0u;
    const bool leader_cta = cta_rank == 0;

    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int i = 0; i < kStages; ++i) {
            // K block i may be multiplied when its operands are there (the A loader and the B loader of every CTA) and its accumulator has been
            // read (lane 0 of every summing warp, when it has taken K block i - kAccums): one barrier, one wait of the MMA issuer.
            mbar_init(full_bar + i, (2 + kSumWarps) * kCtas);
            mbar_init(empty_bar + i, 1);  // tcgen05.commit of the MMA issuer
        }
        for (int i = 0; i < kAccums; ++i) {
            mbar_init(tmem_full_bar + i, 2);  // tcgen05.commit of the MMA issuer, and this CTA's scale warp: products and scales are there
        }
        fence_mbar_init();
        prefetch_tensormap(&tm_a);
        prefetch_tensormap(&tm_b);
    }
    pdl_prologue();  // everything above touches only this CTA's shared memory and the kernel's own parameters
    if (p.mode == kModePsum || p.mode == kModeMasked) {
        int* tiles_end = table + 2 * kMaxCachedGroups;
        for (int i = threadIdx.x; i < p.num_groups; i += kThreads) {
            int first, count, scaled;
            Sched::group_extent(p, i, first, count, scaled);
            table[i] = first;
            table[kMaxCachedGroups + i] = count;
            table[3 * kMaxCachedGroups + i] = scaled;
            tiles_end[i] = (count + Sched::kTileM - 1) / Sched::kTileM * ((p.n + BLOCK_N - 1) / BLOCK_N);
        }
        __syncthreads();
        if (warp == 0) {
            const int chunk = (p.num_groups + 31) / 32;
            const int lo = min(static_cast<int>(lane) * chunk, p.num_groups), hi = min(lo + chunk, p.num_groups);
            int sum = 0;
            for (int i = lo; i < hi; ++i) sum += tiles_end[i];
            int incl = sum;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, incl, off);
                if (static_cast<int>(lane) >= off) incl += v;
            }
            int run = incl - sum;
            for (int i = lo; i < hi; ++i) {
                run += tiles_end[i];
                tiles_end[i] = run;
            }
        }
    }
    if constexpr (kPair) cluster_sync_all();  // both CTAs run and see each other's initialised barriers
    if (warp == 2) {
        if constexpr (kPair) tmem_alloc_pair(tmem_ptr_smem, 512);
        else tmem_alloc(tmem_ptr_smem, 512);
    }
    tcgen05_fence_before();
    __syncthreads();
    if constexpr (kPair) cluster_sync_all();
    tcgen05_fence_after();
    const uint32_t tmem_base = *tmem_ptr_smem;
    // this CTA's K blocks; parts are whole groups of kScaleKb, and the host leaves none empty
    const int tile_ctas = kPair ? 2 : (kSplitK ? static_cast<int>(cluster_num_ctas()) : 1);
    int first_kb = 0, num_kb = (p.k + 127) / 128;  // [first_kb, num_kb)
    if constexpr (kSplitK) {
        const int rank = static_cast<int>(cluster_cta_rank()), units = (num_kb + kScaleKb - 1) / kScaleKb;
        first_kb = units * rank / tile_ctas * kScaleKb;
        num_kb = min(units * (rank + 1) / tile_ctas * kScaleKb, num_kb);
    }

    // In a pair the leader's loaders announce the bytes of both CTAs (their loads are alike), the other CTA's only arrive.
    auto stage_arrive = [&](uint32_t stage, uint32_t bytes) {
        if constexpr (kPair) {
            if (leader_cta) mbar_arrive_expect_tx(full_bar + stage, 2 * bytes);
            else mbar_arrive_cluster(map_to_cta(smem_u32(full_bar + stage), 0));
        } else {
            mbar_arrive_expect_tx(full_bar + stage, bytes);
        }
    };
    auto load_tile = [&](int smem_off, const CUtensorMap* map, uint32_t stage, int x, int y, int z) {
        if constexpr (kPair) tma_load_3d_pair(smem + smem_off, map, map_to_cta(smem_u32(full_bar + stage), 0), x, y, z);
        else tma_load_3d(smem + smem_off, map, full_bar + stage, x, y, z);
    };

    if (warp < 4) {
        setmaxnreg_dec<kRegsBsControl>();
        if (warp == 0 || warp == 3) {
            // ------------------------------------------------------------ loaders: A (warp 0) and B (warp 3)
            const bool is_a = warp == 0;
            const bool elected = elect_one();
            Sched sched(p, table, tile_ctas);
            BlockScaledTile t;
            uint32_t stage = 0, phase = 0;
            bool ok = true;
            while (ok && sched.next(t)) {
                if (t.group < 0) continue;
                const int a_loads = kPair ? 1 : (t.rows + p.a_box_rows - 1) / p.a_box_rows;
                for (int kb = first_kb; kb < num_kb; ++kb) {
                    ok = mbar_wait(empty_bar + stage, phase ^ 1, abort_flag, kTimeoutEmpty, kb);
                    if (!ok) break;
                    if (elected) {
                        if (is_a) {
                            stage_arrive(stage, static_cast<uint32_t>(a_loads * p.a_box_rows) * 128);
                            for (int i = 0; i < a_loads; ++i)
                                load_tile(L::kOffA + stage * L::kABytes + i * p.a_box_rows * 128, &tm_a, stage, kb * 128, t.row0 + i * p.a_box_rows,
                                          p.mode == kModeMasked ? t.group : 0);
                        } else {
                            stage_arrive(stage, L::kBBytes);
                            const int off = L::kOffB + stage * L::kBBytes;
                            const int n = t.n0 + static_cast<int>(cta_rank) * (BLOCK_N / kCtas);  // first channel of this CTA
                            if (BLOCK_N >= 128 && p.b_mn_major) {
#pragma unroll
                                for (int h = 0; h < BLOCK_N / kCtas / 128; ++h)  // boxes of 128 channels x 128 K rows
                                    load_tile(off + h * 16384, &tm_b, stage, n + h * 128, kb * 128, t.group);
                            } else {
                                load_tile(off, &tm_b, stage, kb * 128, n, t.group);
                            }
                        }
                    }
                    __syncwarp();
                    if (++stage == kStages) { stage = 0; phase ^= 1; }
                }
            }
        } else if (warp == 1 && leader_cta) {
            // ------------------------------------------------------------ MMA issuer: one accumulator per K block
            // The summing warps leave this one few issue slots, and a K block is only 512 cycles (256 for a 128-wide tile) of MMAs: its loop holds
            // few instructions. Descriptors are one word each, moved on by additions, and there is one barrier to wait for.
            const bool elected = elect_one();
            Sched sched(p, table, tile_ctas);
            BlockScaledTile t;
            const bool b_mn = BLOCK_N >= 128 && p.b_mn_major;
            const uint32_t idesc = make_idesc_e4m3_f32(128 * kCtas, BLOCK_N) | (b_mn ? (1u << 16) : 0u);
            const uint32_t a_first = desc_lo(smem_u32(smem + L::kOffA), false), b_first = desc_lo(smem_u32(smem + L::kOffB), b_mn);
            const uint32_t b_step = b_mn ? 256u : 2u;  // 32 K rows of 128 bytes, or 32 bytes inside the swizzle span
            uint32_t stage = 0, phase = 0, as = 0;
            uint32_t a_lo = a_first, b_lo = b_first;
            bool ok = true;
            while (ok && sched.next(t)) {
                if (t.group < 0) continue;
#pragma unroll 1
                for (int kb = first_kb; kb < num_kb; ++kb) {
                    ok = mbar_wait(full_bar + stage, phase, abort_flag, kTimeoutFull, kb);
                    if (!ok) break;
                    tcgen05_fence_after();
                    if (elected) {
                        mma_k_block<kPair>(tmem_base + as * kAccumCols, a_lo, b_lo, b_step, idesc);
                        if constexpr (kPair) {
                            tcgen05_commit_pair(tmem_full_bar + as, 3);
                            tcgen05_commit_pair(empty_bar + stage, 3);
                        } else {
                            tcgen05_commit(tmem_full_bar + as);
                            tcgen05_commit(empty_bar + stage);
                        }
                    }
                    __syncwarp();
                    as = as + 1 == kAccums ? 0 : as + 1;
                    a_lo += L::kABytes >> 4;
                    b_lo += L::kBBytes >> 4;
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1;
                        a_lo = a_first;
                        b_lo = b_first;
                    }
                }
            }
        } else if (warp == 2) {
            // ------------------------------------------------------------ scales: sfa[row] * sfb[column block]
            // The loads of four K blocks are under way together, well ahead of their use; read by the summing warps
            // themselves, one K block ahead, their latency was a fifth of the kernel.
            Sched sched(p, table, tile_ctas);
            BlockScaledTile t;
            uint32_t as = 0, phase = 0, slot = 0;
            bool ok = true;
            while (ok && sched.next(t)) {
                if (t.group < 0) continue;
                const long long group = t.group;
                // rows with scales: padding rows that are stored have none (a zero there keeps what their words hold out of d)
                const int scaled_rows = p.store_padding ? min(t.rows, table[3 * kMaxCachedGroups + t.group] - t.row0) : t.rows;
                const float* sfa = p.sfa + (p.mode == kModeMasked ? group * p.sfa_group_stride : 0) + static_cast<long long>(t.row0 + static_cast<int>(lane)) * p.sfa_row_stride;
                // B's scales are the same for all rows: lane 4 h + i loads the one of half h and K block i of the four
                const float* sfb = p.sfb + group * p.sfb_group_stride +
                                   static_cast<long long>(min(t.n0 + static_cast<int>(lane / kScaleKb % 2) * (BLOCK_N / 2), p.n - 1) / 128) * p.sfb_n_stride +
                                   (lane % kScaleKb) * p.sfb_k_stride;
                for (int kb = first_kb; ok && kb < num_kb; kb += kScaleKb) {
                    float a[4][kScaleKb];
                    const bool whole = p.sf_vec && kb + kScaleKb <= num_kb;
#pragma unroll
                    for (int j = 0; j < 4; ++j)  // rows that are not stored need no scale: none is read for them
                        load_scales(sfa + 32 * j * p.sfa_row_stride + kb * p.sfa_k_stride, p.sfa_k_stride,
                                    static_cast<int>(lane) + 32 * j < scaled_rows ? num_kb - kb : 0, whole, a[j]);
                    const float b = static_cast<int>(lane % kScaleKb) < num_kb - kb ? __ldg(sfb + kb * p.sfb_k_stride) : 0.0f;
#pragma unroll
                    for (int i = 0; i < kScaleKb; ++i) {
                        if (!ok || kb + i >= num_kb) break;
                        ok = mbar_wait(tmem_full_bar + as, phase ^ 1, abort_flag, kTimeoutTmemFull, kb);  // K block kb + i - kAccums
                        if (!ok) break;
                        float* to = reinterpret_cast<float*>(smem + L::kOffScales + slot * L::kScaleSlotBytes) + lane;
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float bh = __shfl_sync(0xffffffffu, b, h * kScaleKb + i);
#pragma unroll
                            for (int j = 0; j < 4; ++j) to[h * 128 + 32 * j] = a[j][i] * bh;
                        }
                        __syncwarp();
                        if (lane == 0) mbar_arrive(tmem_full_bar + as);
                        if (++as == kAccums) { as = 0; phase ^= 1; }
                        if (++slot == L::kScaleSlots) slot = 0;
                    }
                }
            }
        }
    } else {
        setmaxnreg_inc<kRegsBsSum>();
        // ---------------------------------------------------------------- running sums and epilogue
        const uint32_t q = warp & 3, half = (warp - 4) >> 2;  // lane quarter of tensor memory, half of the tile's columns
        const int r = static_cast<int>(q * 32 + lane);
        uint8_t* stage_buf = smem + L::kOffStage + (warp - 4) * L::kStagingBytes;
        // the barriers of the MMA issuer's CTA
        const uint32_t issuer_full = kPair ? map_to_cta(smem_u32(full_bar), 0) : smem_u32(full_bar);
        auto give_accumulator = [&](uint32_t to_stage) {
            if constexpr (kPair) mbar_arrive_cluster(issuer_full + to_stage * 8);
            else mbar_arrive(full_bar + to_stage);
        };
        static_assert(kAccums <= kStages, "a K block's barrier is past its previous use when its accumulator is given back");
        if (lane == 0) {
            for (int i = 0; i < kAccums; ++i) give_accumulator(i);  // all are free
        }
        const uint32_t tmem_half = tmem_base + ((q * 32u) << 16) + half * kCols;
        const float* const my_scales = reinterpret_cast<const float*>(smem + L::kOffScales) + half * 128 + r;
        Sched sched(p, table, tile_ctas);
        BlockScaledTile t;
        // K blocks so far, and the stage of the one that will use the accumulator at hand next (kAccums K blocks later)
        uint32_t it = 0, next_stage = kAccums % kStages;
        bool ok = true;
        while (ok && sched.next(t)) {
            if (t.group < 0) continue;
            const bool warp_has_rows = static_cast<int>(q * 32) < t.rows;
            if constexpr (kF32) {
                // c on its way into L2 while the tile is multiplied: all SMs ask for it at once at the end
                if (p.c != nullptr && r < t.rows) {
                    const int col = t.n0 + static_cast<int>(half) * kCols;
                    const float* c = p.c + static_cast<long long>(t.row0 + r) * p.c_row_stride + col;
                    for (int i = 0; i < kCols && col + i < p.n; i += 32) prefetch_l2(c + i);
                }
            }
            float acc[kCols];
#pragma unroll
            for (int i = 0; i < kCols; ++i) acc[i] = 0.0f;
// twice: the jump back costs an instruction fetch (8192 x 7168 x 4096 on pairs 226 -> 216 us)
#pragma unroll 2
            for (int kb = first_kb; kb < num_kb; ++kb) {
                const uint32_t as = it % kAccums;
                ok = mbar_wait(tmem_full_bar + as, (it / kAccums) & 1, abort_flag, kTimeoutTmemFull, kb);
                if (!ok) break;
                tcgen05_fence_after();
                if (warp_has_rows) {
                    constexpr int kChunk = 16;  // columns per load; the next load is under way while a chunk is added
                    const uint32_t tmem_row = tmem_half + as * kAccumCols;
                    uint32_t v[2][kChunk];
                    tmem_ld_32x32b_x16(tmem_row, v[0]);
                    const float s = my_scales[(it % L::kScaleSlots) * (L::kScaleSlotBytes / 4)];
#pragma unroll
                    for (int c = 0; c < kCols / kChunk; ++c) {
                        tmem_ld_wait();
                        if (c + 1 < kCols / kChunk) tmem_ld_32x32b_x16(tmem_row + (c + 1) * kChunk, v[(c + 1) & 1]);
#pragma unroll
                        for (int i = 0; i < kChunk; i += 2) fma_f32x2(acc[c * kChunk + i], acc[c * kChunk + i + 1], v[c & 1][i], v[c & 1][i + 1], s);
                    }
                }
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) {
                    give_accumulator(next_stage);                  // this warp has read the accumulator (and the scales)
                }
                ++it;
                if (++next_stage == kStages) next_stage = 0;
            }
            if (!ok) break;
            if (!warp_has_rows) continue;
            if constexpr (kSplitK) {
                // All MMAs of this CTA are complete and with them its loads: the ring is free. 16-byte chunks, XOR-swizzled.
                uint8_t* mine = smem + r * (BLOCK_N * 4);
#pragma unroll
                for (int i = 0; i < kCols / 4; ++i)
                    *reinterpret_cast<float4*>(mine + (((static_cast<int>(half) * (kCols / 4) + i) ^ (r & 7)) << 4)) =
                        make_float4(acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3]);
                continue;  // the cluster adds and stores below
            }
            const int col0 = t.n0 + static_cast<int>(half) * kCols;
            // Store: 16 rows x 128 bytes at a time are turned through shared memory (16-byte chunks, XOR-swizzled): the rows' 16 lanes write them,
            // then every store instruction of the warp writes four whole lines instead of 16 bytes of 32 rows.
            constexpr int kPerChunk = kF32 ? 4 : 8;                              // columns in 16 bytes
            constexpr int kChunks = kCols / kPerChunk < 8 ? kCols / kPerChunk : 8;  // of a row of the slab
            constexpr int kSlab = kChunks * kPerChunk;
            auto place = [&](int row, int chunk) { return reinterpret_cast<uint4*>(stage_buf + row * 128 + ((chunk ^ (row & (kChunks - 1))) << 4)); };
            const long long row_base = (p.mode == kModeMasked ? static_cast<long long>(t.group) * p.m : 0) + t.row0 + static_cast<int>(q * 32);
            const int rows_here = t.rows - static_cast<int>(q * 32);
#pragma unroll
            for (int s = 0; s < kCols / kSlab; ++s) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (h * 16 >= rows_here) continue;
                    __syncwarp();
                    if (static_cast<int>(lane >> 4) == h) {
#pragma unroll
                        for (int i = 0; i < kChunks; ++i) {
                            const float* a = acc + s * kSlab + i * kPerChunk;
                            if constexpr (kF32)
                                *place(lane & 15, i) = make_uint4(__float_as_uint(a[0]), __float_as_uint(a[1]), __float_as_uint(a[2]), __float_as_uint(a[3]));
                            else
                                *place(lane & 15, i) = make_uint4(pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3]), pack_bf16x2(a[4], a[5]), pack_bf16x2(a[6], a[7]));
                        }
                    }
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < kChunks / 2; ++j) {
                        constexpr int kRowsPer = 32 / kChunks;
                        const int row = static_cast<int>(lane) / kChunks + kRowsPer * j, chunk = static_cast<int>(lane) % kChunks;
                        const int col = col0 + s * kSlab + chunk * kPerChunk;
                        if (h * 16 + row >= rows_here || col >= p.n) continue;  // n is a multiple of 8: a chunk is inside or outside
                        const uint4 v = *place(row, chunk);
                        const long long at = (row_base + h * 16 + row) * p.d_row_stride + col;
                        if constexpr (kF32) {
                            float4 f = make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
                            if (p.c != nullptr) {
                                const float4 c4 = *reinterpret_cast<const float4*>(p.c + (row_base + h * 16 + row) * p.c_row_stride + col);
                                f = make_float4(c4.x + f.x, c4.y + f.y, c4.z + f.z, c4.w + f.w);
                            }
                            *reinterpret_cast<float4*>(static_cast<float*>(p.d) + at) = f;
                        } else {
                            st_global_v4(static_cast<__nv_bfloat16*>(p.d) + at, v.x, v.y, v.z, v.w);
                        }
                    }
                }
            }
        }
    }

    if constexpr (kSplitK) {
        // A CTA that gave up on a wait leaves zeros or stale bytes in its part; the error is in the status block.
        __syncwarp();
        cluster_sync_all();
        Sched sched(p, table, tile_ctas);
        BlockScaledTile t;
        if (sched.next(t)) {
            constexpr int kOct = BLOCK_N / 8;  // 8 columns per thread and step
            const int items = max(t.rows, 0) * kOct;
            for (int i = static_cast<int>(cluster_cta_rank() * kGemmThreads + threadIdx.x); i < items; i += tile_ctas * kGemmThreads) {
                const int row = i / kOct, oct = i % kOct, col = t.n0 + oct * 8;
                if (col >= p.n) continue;
                const uint32_t at_row = smem_u32(smem + row * (BLOCK_N * 4));
                float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                for (int c0 = 0; c0 < tile_ctas; c0 += 2) {  // two ranks' loads in flight
                    float4 f[2][2];
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            f[c][h] = ld_cluster_f4(map_to_cta(at_row + (((oct * 2 + h) ^ (row & 7)) << 4), static_cast<uint32_t>(c0 + c)));
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            v[4 * h] += f[c][h].x;
                            v[4 * h + 1] += f[c][h].y;
                            v[4 * h + 2] += f[c][h].z;
                            v[4 * h + 3] += f[c][h].w;
                        }
                }
                const long long at = static_cast<long long>(t.row0 + row) * p.d_row_stride + col;
                if constexpr (kF32) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float4 o = make_float4(v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]);
                        if (p.c != nullptr) {
                            const float4 c4 = *reinterpret_cast<const float4*>(p.c + static_cast<long long>(t.row0 + row) * p.c_row_stride + col + 4 * h);
                            o = make_float4(c4.x + o.x, c4.y + o.y, c4.z + o.z, c4.w + o.w);
                        }
                        *reinterpret_cast<float4*>(static_cast<float*>(p.d) + at + 4 * h) = o;
                    }
                } else {
                    st_global_v4(static_cast<__nv_bfloat16*>(p.d) + at, pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                                 pack_bf16x2(v[6], v[7]));
                }
            }
        }
        cluster_sync_all();  // nobody leaves while others read its shared memory
    }

    // ---------------------------------------------------------------- teardown
    tcgen05_fence_before();
    __syncthreads();
    if (*abort_flag != 0) {
        // Let copies and MMAs that were already issued land before shared and tensor memory are released.
        __nanosleep(100000);
        __syncthreads();
    }
    if constexpr (kPair) cluster_sync_all();  // the other CTA may still signal barriers of this one or read its shared memory
    if (warp == 2) {
        tcgen05_fence_after();
        if constexpr (kPair) tmem_dealloc_pair(tmem_base, 512);
        else tmem_dealloc(tmem_base, 512);
    }
}

}  // namespace dgb
