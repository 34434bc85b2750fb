// Tokens sorted by expert and back, as operators of their own: the dispatch plan (a stable sort of the (token, k) entries by
// expert), the permutation of token rows into expert order, the weighted sum back, and the gradients of both. The layers do
// the same inside their calls (moe_kernels.cuh); these serve callers that run the grouped GEMMs themselves, a training step above
// all. Everything here is bound by HBM, small batches by launches and latency; no atomics touch global memory, so every result is the same in every run.
#pragma once

#include <cuda_bf16.h>

#include "ptx.cuh"

namespace dgb {

constexpr int kPlanThreads = 1024;
constexpr int kMaxPlanExperts = 1024;

// Experts counted per chunk of entries: chunk_hist[chunk][e]. (The end of the last chunk, rounded up, stays below 2^31: the host sees to it.)
__global__ void __launch_bounds__(kPlanThreads)
dgb200_sort_count_kernel(const long long* __restrict__ topk_idx, int entries, int chunk_entries, int experts, int* __restrict__ chunk_hist) {
    pdl_prologue();
    __shared__ int hist[kMaxPlanExperts];
    for (int e = threadIdx.x; e < experts; e += kPlanThreads) hist[e] = 0;
    __syncthreads();
    const int lo = blockIdx.x * chunk_entries, hi = min(lo + chunk_entries, entries);
    for (int i = lo + static_cast<int>(threadIdx.x); i < hi; i += kPlanThreads) {
        const long long e = topk_idx[i];
        if (e >= 0 && e < experts) atomicAdd(&hist[e], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < experts; e += kPlanThreads) chunk_hist[static_cast<long long>(blockIdx.x) * experts + e] = hist[e];
}

// dest_row[entry] = first row of its expert + entries of the same expert before it (-1: masked, or not one of the experts);
// expert_start / expert_end = the experts' segments, each starting at a multiple of `alignment`. Every CTA derives the
// segments of all experts and its own chunk's offsets from the chunks' counts (a thread per expert, the loads independent), which
// takes less than a launch of its own would. chunk_hist null: one CTA, which counts its entries itself.
__global__ void __launch_bounds__(kPlanThreads)
dgb200_sort_assign_kernel(const long long* __restrict__ topk_idx, int entries, int chunk_entries, int experts, int alignment,
                          const int* __restrict__ chunk_hist, int* __restrict__ dest_row, int* __restrict__ expert_start,
                          int* __restrict__ expert_end) {
    pdl_prologue();
    extern __shared__ unsigned char warp_hist[];  // [32 warps][experts]: a warp's entries of each expert, at most 32
    __shared__ int next_row[kMaxPlanExperts];
    __shared__ int warp_sums[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int e = static_cast<int>(threadIdx.x);  // the expert of this thread
    int before = 0, count = 0;
    if (chunk_hist != nullptr) {
        if (e < experts) {
            const int chunks = static_cast<int>(gridDim.x);
#pragma unroll 8
            for (int c = 0; c < chunks; ++c) {
                const int v = __ldg(chunk_hist + static_cast<long long>(c) * experts + e);
                count += v;
                if (c < static_cast<int>(blockIdx.x)) before += v;
            }
        }
    } else {
        next_row[e] = 0;
        __syncthreads();
        for (int i = e; i < entries; i += kPlanThreads) {
            const long long x = topk_idx[i];
            if (x >= 0 && x < experts) atomicAdd(&next_row[x], 1);
        }
        __syncthreads();
        count = next_row[e];
    }
    const int padded = (count + alignment - 1) / alignment * alignment;
    int incl = padded;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += v;
    }
    if (lane == 31) warp_sums[warp] = incl;
    __syncthreads();
    if (warp == 0) {
        int w = warp_sums[lane];
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, w, off);
            if (lane >= off) w += v;
        }
        warp_sums[lane] = w;
    }
    __syncthreads();
    const int start = (warp > 0 ? warp_sums[warp - 1] : 0) + incl - padded;
    next_row[e] = start + before;
    if (blockIdx.x == 0 && e < experts) {
        expert_start[e] = start;
        expert_end[e] = start + count;
    }
    const int lo = blockIdx.x * chunk_entries, hi = min(lo + chunk_entries, entries);
    for (int base = lo; base < hi; base += kPlanThreads) {
        for (int i = e; i < 8 * experts; i += kPlanThreads) reinterpret_cast<unsigned*>(warp_hist)[i] = 0;
        __syncthreads();
        const int i = base + static_cast<int>(threadIdx.x);
        int mine = -1;
        if (i < hi) {
            const long long x = topk_idx[i];
            if (x >= 0 && x < experts) mine = static_cast<int>(x);
        }
        const unsigned peers = __match_any_sync(0xffffffffu, mine);
        const int rank = __popc(peers & ((1u << lane) - 1u));
        if (mine >= 0 && rank == 0) warp_hist[warp * experts + mine] = static_cast<unsigned char>(__popc(peers));
        __syncthreads();
        if (i < hi) {
            int dest = -1;
            if (mine >= 0) {
                dest = next_row[mine] + rank;
                for (int w = 0; w < warp; ++w) dest += warp_hist[w * experts + mine];
            }
            dest_row[i] = dest;
        }
        __syncthreads();
        if (base + kPlanThreads < hi) {
            int sum = 0;
            if (e < experts)
                for (int w = 0; w < 32; ++w) sum += warp_hist[w * experts + e];
            __syncthreads();
            next_row[e] += sum;
        }
    }
}

// The whole plan of a small batch (at most 1024 entries) in one CTA of as many threads as there are entries or experts: every entry is read
// once and ranked within its warp, a thread per expert adds up the warps. 104 entries, 256 experts: 2.2 us where calls follow each other (the
// kernels below read the entries twice and count with atomics, about 4).
__global__ void __launch_bounds__(kPlanThreads)
dgb200_sort_small_kernel(const long long* __restrict__ topk_idx, int entries, int experts, int alignment, int* __restrict__ dest_row,
                         int* __restrict__ expert_start, int* __restrict__ expert_end) {
    pdl_prologue();
    extern __shared__ unsigned char warp_hist[];  // [warps with entries][experts], padded to words
    __shared__ int first_row[kMaxPlanExperts];
    __shared__ int warp_sums[32];
    const int i = static_cast<int>(threadIdx.x), lane = i & 31, warp = i >> 5;
    const int used = (entries + 31) / 32, row_bytes = (experts + 3) / 4 * 4;
    int mine = -1;
    if (i < entries) {
        const long long x = topk_idx[i];
        if (x >= 0 && x < experts) mine = static_cast<int>(x);
    }
    for (int w = i; w < used * row_bytes / 4; w += blockDim.x) reinterpret_cast<unsigned*>(warp_hist)[w] = 0;
    if (i < 32) warp_sums[i] = 0;
    __syncthreads();
    const unsigned peers = __match_any_sync(0xffffffffu, mine);
    const int rank = __popc(peers & ((1u << lane) - 1u));
    if (mine >= 0 && rank == 0) warp_hist[warp * row_bytes + mine] = static_cast<unsigned char>(__popc(peers));
    __syncthreads();
    int count = 0;
    if (i < experts)
        for (int w = 0; w < used; ++w) count += warp_hist[w * row_bytes + i];
    const int padded = (count + alignment - 1) / alignment * alignment;
    int incl = padded;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += v;
    }
    if (lane == 31) warp_sums[warp] = incl;
    __syncthreads();
    int start = incl - padded;
    for (int w = 0; w < warp; ++w) start += warp_sums[w];
    if (i < experts) {
        first_row[i] = start;
        expert_start[i] = start;
        expert_end[i] = start + count;
    }
    __syncthreads();
    if (i >= entries) return;
    int dest = -1;
    if (mine >= 0) {
        dest = first_row[mine] + rank;
        for (int w = 0; w < warp; ++w) dest += warp_hist[w * row_bytes + mine];
    }
    dest_row[i] = dest;
}

// Rows of one tensor on their way to expert order (a second tensor, the rows' scale factors, may go along).
struct PermuteRows {
    const unsigned char* from;  // [tokens] rows
    unsigned char* to;          // [capacity] rows
    long long from_stride, to_stride;  // bytes
    long long row_vecs;         // vectors of the row
};

struct PermuteParams {
    PermuteRows rows, scales;  // scales.from null: none
    const int* dest_row;
    const int* expert_end;
    int tokens, topk, experts, alignment, capacity;
    int column_blocks;   // CTAs that share a token's row
    int padding_blocks;  // CTAs per expert that zero its padding rows, 8 rows each (0: padding rows are left as they are)
};

// The rows of a token's entries into shared memory (-1: masked). A row that the buffer does not hold is reported and left out.
__device__ __forceinline__ void load_entries(const int* dest_row, const float* weights, int token, int topk, int capacity, int* dest, float* weight) {
    if (static_cast<int>(threadIdx.x) < topk) {
        const long long at = static_cast<long long>(token) * topk + threadIdx.x;
        const int row = dest_row[at];
        if (row >= capacity) report_error(kBadArgument, row, capacity);
        const bool used = row >= 0 && row < capacity;
        dest[threadIdx.x] = used ? row : -1;
        if (weight != nullptr) weight[threadIdx.x] = used && weights != nullptr ? weights[at] : 1.0f;
    }
    __syncthreads();
}

// Row of padding that this warp zeroes, or -1: the CTAs behind the tokens' take 8 rows of an expert's padding each.
__device__ __forceinline__ long long padding_row(const int* expert_end, int block, int blocks_per_expert, int alignment, int capacity) {
    const int e = block / blocks_per_expert;
    const int end = __ldg(expert_end + e);
    const long long row = end + (block - e * blocks_per_expert) * 8ll + (threadIdx.x >> 5);
    const long long aligned_end = (static_cast<long long>(end) + alignment - 1) / alignment * alignment;
    return end >= 0 && row < aligned_end && row < capacity ? row : -1;
}

template <typename Vec>
__device__ __forceinline__ void scatter_row(const PermuteRows& r, int token, const int* dest, int topk, int lane0, int step) {
    const Vec* from = reinterpret_cast<const Vec*>(r.from + token * r.from_stride);
    for (long long c0 = lane0; c0 < r.row_vecs; c0 += 4ll * step) {
        Vec v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (c0 + j * step < r.row_vecs) v[j] = __ldg(from + c0 + j * step);
        for (int k = 0; k < topk; ++k) {
            const int row = dest[k];
            if (row < 0) continue;
            Vec* to = reinterpret_cast<Vec*>(r.to + row * r.to_stride);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c0 + j * step < r.row_vecs) to[c0 + j * step] = v[j];
        }
    }
}

template <typename Vec>
__device__ __forceinline__ void zero_row(const PermuteRows& r, long long row, int lane) {
    Vec* to = reinterpret_cast<Vec*>(r.to + row * r.to_stride);
    for (long long c = lane; c < r.row_vecs; c += 32) to[c] = Vec{};
}

// rows[dest_row[t, k]] = x[t]; padding rows between a segment's end and its aligned end = 0; the rows behind the last segment are left
// as they are. HBM writes bound it: a token's row is read once, held in registers and written topk times. 4099 tokens x 7168 x 8 into 256
// segments of multiples of 128 rows, 528 MB and 257 MB of zeros, with the plan before it and the gradient (530 MB) behind it: 186 us, 7.0
// TB/s of all that moves (some of it stays in L2). The first tokens * column_blocks CTAs: a token's row, or
// a part of its columns; the CTAs behind them: 8 padding rows of an expert, one warp each.
template <typename Vec, typename ScaleVec>
__global__ void __launch_bounds__(256) dgb200_permute_kernel(const PermuteParams p) {
    pdl_prologue();
    const int token_ctas = p.tokens * p.column_blocks;
    if (static_cast<int>(blockIdx.x) < token_ctas) {
        const int token = static_cast<int>(blockIdx.x) / p.column_blocks;
        __shared__ int dest[32];
        load_entries(p.dest_row, nullptr, token, p.topk, p.capacity, dest, nullptr);
        const int lane0 = (static_cast<int>(blockIdx.x) - token * p.column_blocks) * 256 + static_cast<int>(threadIdx.x), step = p.column_blocks * 256;
        scatter_row<Vec>(p.rows, token, dest, p.topk, lane0, step);
        if (p.scales.from != nullptr) scatter_row<ScaleVec>(p.scales, token, dest, p.topk, lane0, step);
        return;
    }
    const long long row = padding_row(p.expert_end, static_cast<int>(blockIdx.x) - token_ctas, p.padding_blocks, p.alignment, p.capacity);
    if (row < 0) return;
    zero_row<Vec>(p.rows, row, threadIdx.x & 31);
    if (p.scales.from != nullptr) zero_row<ScaleVec>(p.scales, row, threadIdx.x & 31);
}

// A vector of kVec values as floats and back (one rounding, to nearest even).
template <typename T, int kVec>
struct RowVec;
template <>
struct RowVec<__nv_bfloat16, 8> {
    using Raw = uint4;
    static __device__ __forceinline__ void unpack(const Raw& r, float* f) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ Raw pack(const float* f) {
        return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
    }
};
template <>
struct RowVec<__nv_bfloat16, 1> {
    using Raw = unsigned short;
    static __device__ __forceinline__ void unpack(const Raw& r, float* f) { f[0] = __uint_as_float(static_cast<uint32_t>(r) << 16); }
    static __device__ __forceinline__ Raw pack(const float* f) { return static_cast<Raw>(pack_bf16x2(f[0], 0.0f) & 0xffffu); }
};
template <>
struct RowVec<float, 4> {
    using Raw = float4;
    static __device__ __forceinline__ void unpack(const Raw& r, float* f) { f[0] = r.x, f[1] = r.y, f[2] = r.z, f[3] = r.w; }
    static __device__ __forceinline__ Raw pack(const float* f) { return make_float4(f[0], f[1], f[2], f[3]); }
};
template <>
struct RowVec<float, 1> {
    using Raw = float;
    static __device__ __forceinline__ void unpack(const Raw& r, float* f) { f[0] = r; }
    static __device__ __forceinline__ Raw pack(const float* f) { return f[0]; }
};

struct UnpermuteParams {
    const void* rows;           // [capacity, hidden]
    const void* dy;             // [tokens, hidden], backward only
    void* out;                  // forward: y [tokens, hidden]; backward: d_rows [capacity, hidden]
    float* d_weights;           // [tokens, topk], backward only
    const float* weights;       // [tokens, topk], or null: 1
    const int* dest_row;
    const int* expert_end;      // backward only
    long long rows_stride, dy_stride, out_stride;  // elements
    int tokens, topk, hidden, experts, alignment, capacity, padding_blocks;
};

// y[t] = sum over k of weights[t, k] rows[dest_row[t, k]], in ascending k in FP32, rounded once; a masked entry adds nothing (its weight
// is not read). Without weights it is the gradient of the permutation. HBM reads bound it; eight rows' loads are in flight per
// thread (4096 tokens x 4096 x 8, cold: 269 MB read in 51 us).
template <typename T, int kVec>
__global__ void __launch_bounds__(128) dgb200_unpermute_kernel(const UnpermuteParams p) {
    using V = RowVec<T, kVec>;
    using Raw = typename V::Raw;
    pdl_prologue();
    __shared__ int dest[32];
    __shared__ float weight[32];
    const int token = static_cast<int>(blockIdx.x);
    load_entries(p.dest_row, p.weights, token, p.topk, p.capacity, dest, weight);
    const T* rows = static_cast<const T*>(p.rows);
    T* out = static_cast<T*>(p.out) + token * p.out_stride;
    for (int c = (blockIdx.y * 128 + threadIdx.x) * kVec; c < p.hidden; c += gridDim.y * 128 * kVec) {
        float acc[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i) acc[i] = 0.0f;
        for (int k0 = 0; k0 < p.topk; k0 += 8) {
            Raw raw[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (k0 + j < p.topk && dest[k0 + j] >= 0) raw[j] = __ldg(reinterpret_cast<const Raw*>(rows + dest[k0 + j] * p.rows_stride + c));
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (k0 + j < p.topk && dest[k0 + j] >= 0) {
                    float f[kVec];
                    V::unpack(raw[j], f);
                    const float w = weight[k0 + j];
#pragma unroll
                    for (int i = 0; i < kVec; ++i) acc[i] = fmaf(w, f[i], acc[i]);
                }
        }
        *reinterpret_cast<Raw*>(out + c) = V::pack(acc);
    }
}

// The gradients of the weighted sum: d_rows[dest_row[t, k]] = weights[t, k] dy[t], d_weights[t, k] = <rows[dest_row[t, k]], dy[t]> (0 for a
// masked entry); padding rows of d_rows = 0, as the K-grouped GEMM wants them, rows behind the last segment stay. One CTA per token: dy is
// read once a batch of eight entries, the dot products are summed in a fixed order (thread, warp, CTA). HBM bounds it; with 76 registers
// three CTAs a SM kept too little in flight (8192 tokens x 4096 x 8, forward and backward: 283 us, with four, which spill two words of the
// BF16 form, 275, its bytes at the copy rate 272).
template <typename T, int kVec>
__global__ void __launch_bounds__(256, 4) dgb200_unpermute_backward_kernel(const UnpermuteParams p) {
    using V = RowVec<T, kVec>;
    using Raw = typename V::Raw;
    pdl_prologue();
    T* out = static_cast<T*>(p.out);
    if (static_cast<int>(blockIdx.x) >= p.tokens) {
        const long long row = padding_row(p.expert_end, static_cast<int>(blockIdx.x) - p.tokens, p.padding_blocks, p.alignment, p.capacity);
        if (row < 0) return;
        for (int c = (threadIdx.x & 31) * kVec; c < p.hidden; c += 32 * kVec) *reinterpret_cast<Raw*>(out + row * p.out_stride + c) = Raw{};
        return;
    }
    __shared__ int dest[32];
    __shared__ float weight[32];
    __shared__ float partial[8][32];
    const int token = static_cast<int>(blockIdx.x);
    load_entries(p.dest_row, p.weights, token, p.topk, p.capacity, dest, weight);
    const T* rows = static_cast<const T*>(p.rows);
    const T* dy = static_cast<const T*>(p.dy) + token * p.dy_stride;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int k0 = 0; k0 < p.topk; k0 += 8) {
        float dot[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        for (int c = threadIdx.x * kVec; c < p.hidden; c += 256 * kVec) {
            float g[kVec];
            V::unpack(__ldg(reinterpret_cast<const Raw*>(dy + c)), g);
            Raw raw[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (k0 + j < p.topk && dest[k0 + j] >= 0) raw[j] = __ldg(reinterpret_cast<const Raw*>(rows + dest[k0 + j] * p.rows_stride + c));
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (k0 + j < p.topk && dest[k0 + j] >= 0) {
                    float f[kVec], o[kVec];
                    V::unpack(raw[j], f);
                    const float w = weight[k0 + j];
#pragma unroll
                    for (int i = 0; i < kVec; ++i) {
                        dot[j] = fmaf(f[i], g[i], dot[j]);
                        o[i] = w * g[i];
                    }
                    *reinterpret_cast<Raw*>(out + dest[k0 + j] * p.out_stride + c) = V::pack(o);
                }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            for (int off = 16; off > 0; off >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], off);
            if (lane == 0 && k0 + j < p.topk) partial[warp][k0 + j] = dot[j];
        }
    }
    __syncthreads();
    if (static_cast<int>(threadIdx.x) < p.topk) {
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; ++w) sum += partial[w][threadIdx.x];
        p.d_weights[static_cast<long long>(token) * p.topk + threadIdx.x] = sum;
    }
}

}  // namespace dgb
