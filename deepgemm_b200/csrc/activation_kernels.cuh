// SwiGLU of the experts' rows, forward and backward, as operators of their own (the layers fuse the forward form into their
// gate/up GEMM). Rows are [gate | up]; with a clamp c the gate is min(gate, c) and up is clamped to [-c, c], and the
// gradient is zero where a clamp holds. Bound by HBM: every value is read and written once in 16-byte vectors, four rows a thread where
// there are many (32768 x 2 x 2048: forward 60.5 us, 6.65 TB/s; forward and backward over 64 segments 179 us, 36864 rows at most; to FP8 59.4 us,
// 5.7 TB/s, where the issue slots are 76 % taken).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "permute_kernels.cuh"  // RowVec
#include "ptx.cuh"

namespace dgb {

struct SwigluParams {
    const __nv_bfloat16* x;  // [rows, 2 inter]
    const __nv_bfloat16* dy; // [rows, inter], backward only
    void* out;               // BF16 [rows, inter], E4M3 [rows, inter], or BF16 [rows, 2 inter] (backward)
    float* sf;               // FP8 only: [rows, ceil(inter / 128)]
    long long x_stride, dy_stride, out_stride, sf_stride;  // elements
    const int* layout;       // psum layout: only rows below the last group's aligned end; null: all
    int num_groups, alignment, rows, inter;
    float clamp;             // <= 0: none
};

__device__ __forceinline__ int swiglu_rows(const SwigluParams& p) {
    if (p.layout == nullptr) return p.rows;
    const long long end = max(__ldg(p.layout + p.num_groups - 1), 0);
    return static_cast<int>(min((end + p.alignment - 1) / p.alignment * p.alignment, static_cast<long long>(p.rows)));
}

// The clamp passes NaN on, as a comparison does and fminf does not.
__device__ __forceinline__ float clamp_above(float v, float c) { return v > c ? c : v; }
__device__ __forceinline__ float clamp_both(float v, float c) { return v > c ? c : (v < -c ? -c : v); }

// 1 / (1 + e^-x) from the hardware's exponential and reciprocal: about 2^-22 off, far below the BF16 or E4M3 rounding that follows.
__device__ __forceinline__ float sigmoid_fast(float x) { return rcp_approx(1.0f + __expf(-x)); }

// One thread: kVec columns of kRows consecutive rows, so that 2 kRows loads (3 kRows backward) are in flight.
template <int kVec, int kRows>
__global__ void __launch_bounds__(256) dgb200_swiglu_kernel(const SwigluParams p) {
    using V = RowVec<__nv_bfloat16, kVec>;
    using Raw = typename V::Raw;
    pdl_prologue();
    const int rows = swiglu_rows(p);
    const int col = static_cast<int>(blockIdx.y * blockDim.x + threadIdx.x) * kVec;
    const int row0 = static_cast<int>(blockIdx.x) * kRows;
    if (col >= p.inter || row0 >= rows) return;
    Raw gate[kRows], up[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r)
        if (row0 + r < rows) {
            const __nv_bfloat16* x = p.x + (row0 + r) * p.x_stride + col;
            gate[r] = __ldg(reinterpret_cast<const Raw*>(x));
            up[r] = __ldg(reinterpret_cast<const Raw*>(x + p.inter));
        }
#pragma unroll
    for (int r = 0; r < kRows; ++r)
        if (row0 + r < rows) {
            float g[kVec], u[kVec], y[kVec];
            V::unpack(gate[r], g);
            V::unpack(up[r], u);
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                if (p.clamp > 0.0f) {
                    g[i] = clamp_above(g[i], p.clamp);
                    u[i] = clamp_both(u[i], p.clamp);
                }
                y[i] = g[i] * sigmoid_fast(g[i]) * u[i];
            }
            *reinterpret_cast<Raw*>(static_cast<__nv_bfloat16*>(p.out) + (row0 + r) * p.out_stride + col) = V::pack(y);
        }
}

// d_gate = dy u s(g) (1 + g (1 - s(g))), d_up = dy g s(g); zero where the clamp holds.
template <int kVec, int kRows>
__global__ void __launch_bounds__(256) dgb200_swiglu_backward_kernel(const SwigluParams p) {
    using V = RowVec<__nv_bfloat16, kVec>;
    using Raw = typename V::Raw;
    pdl_prologue();
    const int rows = swiglu_rows(p);
    const int col = static_cast<int>(blockIdx.y * blockDim.x + threadIdx.x) * kVec;
    const int row0 = static_cast<int>(blockIdx.x) * kRows;
    if (col >= p.inter || row0 >= rows) return;
    Raw gate[kRows], up[kRows], grad[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r)
        if (row0 + r < rows) {
            const __nv_bfloat16* x = p.x + (row0 + r) * p.x_stride + col;
            gate[r] = __ldg(reinterpret_cast<const Raw*>(x));
            up[r] = __ldg(reinterpret_cast<const Raw*>(x + p.inter));
            grad[r] = __ldg(reinterpret_cast<const Raw*>(p.dy + (row0 + r) * p.dy_stride + col));
        }
#pragma unroll
    for (int r = 0; r < kRows; ++r)
        if (row0 + r < rows) {
            float g[kVec], u[kVec], dy[kVec], dg[kVec], du[kVec];
            V::unpack(gate[r], g);
            V::unpack(up[r], u);
            V::unpack(grad[r], dy);
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                float gc = g[i], uc = u[i];
                if (p.clamp > 0.0f) {
                    gc = clamp_above(gc, p.clamp);
                    uc = clamp_both(uc, p.clamp);
                }
                const float s = sigmoid_fast(gc);
                dg[i] = dy[i] * uc * s * fmaf(gc, 1.0f - s, 1.0f);
                du[i] = dy[i] * gc * s;
                if (p.clamp > 0.0f) {
                    if (g[i] > p.clamp) dg[i] = 0.0f;
                    if (fabsf(u[i]) > p.clamp) du[i] = 0.0f;
                }
            }
            __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out) + (row0 + r) * p.out_stride + col;
            *reinterpret_cast<Raw*>(out) = V::pack(dg);
            *reinterpret_cast<Raw*>(out + p.inter) = V::pack(du);
        }
}

// Forward straight to E4M3 with one FP32 scale per 128 columns (sf = max(amax, 1e-4) / 448, q = e4m3(y / sf)): the products stay in FP32 until
// that one rounding. A lane owns 8 columns, 16 lanes a scale block; inter is a multiple of 8, a last block may be short.
template <int kRows>
__global__ void __launch_bounds__(256) dgb200_swiglu_cast_kernel(const SwigluParams p) {
    using V = RowVec<__nv_bfloat16, 8>;
    pdl_prologue();
    const int rows = swiglu_rows(p);
    const int col = static_cast<int>(blockIdx.y * blockDim.x + threadIdx.x) * 8;
    const int row0 = static_cast<int>(blockIdx.x) * kRows;
    if (row0 >= rows) return;
    const bool inside = col < p.inter;  // lanes outside take part in the shuffles
    uint4 gate[kRows], up[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        gate[r] = up[r] = make_uint4(0, 0, 0, 0);
        if (inside && row0 + r < rows) {
            const __nv_bfloat16* x = p.x + (row0 + r) * p.x_stride + col;
            gate[r] = __ldg(reinterpret_cast<const uint4*>(x));
            up[r] = __ldg(reinterpret_cast<const uint4*>(x + p.inter));
        }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        float g[8], u[8], y[8], amax = 0.0f;
        V::unpack(gate[r], g);
        V::unpack(up[r], u);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (p.clamp > 0.0f) {
                g[i] = clamp_above(g[i], p.clamp);
                u[i] = clamp_both(u[i], p.clamp);
            }
            y[i] = g[i] * sigmoid_fast(g[i]) * u[i];
            amax = fmaxf(amax, fabsf(y[i]));
        }
#pragma unroll
        for (int off = 1; off < 16; off <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
        if (!inside || row0 + r >= rows) continue;
        const float sf = fmaxf(amax, 1e-4f) / 448.0f;
        const float inv = 1.0f / sf;
        const __nv_fp8x4_e4m3 lo(make_float4(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv));
        const __nv_fp8x4_e4m3 hi(make_float4(y[4] * inv, y[5] * inv, y[6] * inv, y[7] * inv));
        *reinterpret_cast<uint2*>(static_cast<unsigned char*>(p.out) + (row0 + r) * p.out_stride + col) = make_uint2(lo.__x, hi.__x);
        if ((threadIdx.x & 15) == 0) p.sf[(row0 + r) * p.sf_stride + col / 128] = sf;
    }
}

}  // namespace dgb
