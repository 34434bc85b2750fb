// SwiGLU of the experts' rows, forward and backward, as operators of their own (the layers fuse the forward form into their
// gate/up GEMM). Rows are [gate | up]; with a clamp c the gate is min(gate, c) and up is clamped to [-c, c], and the
// gradient is zero where a clamp holds. Bound by HBM: every value is read and written once in 16-byte vectors, four rows a thread where
// there are many (32768 x 2 x 2048: forward 60.5 us, 6.65 TB/s; forward and backward over 64 segments 179 us, 36864 rows at most; to FP8 64.5 us,
// 5.2 TB/s, where the issue slots are taken).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "permute_kernels.cuh"  // RowVec
#include "ptx.cuh"
#include "quant_kernels.cuh"   // negated_quotients

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

// 1 / (1 + e^-x) from the hardware's exponential and reciprocal: about 2^-22 off, far below the BF16 rounding that follows.
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

// g u / (1 + e^-g) for two values, as FP32 operations give it: the reciprocal is rounded correctly but for rare cases (one Newton step). An exponent
// past 88 would be infinity times zero in that step; the reciprocal is zero there either way.
__device__ __forceinline__ void swiglu_f32x2(float g0, float g1, float u0, float u1, float& y0, float& y1) {
    const float d0 = 1.0f + expf(fminf(-g0, 88.0f)), d1 = 1.0f + expf(fminf(-g1, 88.0f));
    asm("{\n\t"
        ".reg .b64 g, u, d, r, e, one;\n\t"
        "mov.b64 g, {%2, %3};\n\t"
        "mov.b64 u, {%4, %5};\n\t"
        "mov.b64 d, {%6, %7};\n\t"
        "mov.b64 r, {%8, %9};\n\t"
        "mov.b64 one, {%10, %10};\n\t"
        "fma.rn.f32x2 e, r, d, one;\n\t"
        "fma.rn.f32x2 r, e, r, r;\n\t"
        "mul.rn.f32x2 g, g, r;\n\t"
        "mul.rn.f32x2 g, g, u;\n\t"
        "mov.b64 {%0, %1}, g;\n\t"
        "}\n" : "=f"(y0), "=f"(y1) : "f"(g0), "f"(g1), "f"(u0), "f"(u1), "f"(-d0), "f"(-d1), "f"(rcp_approx(d0)), "f"(rcp_approx(d1)), "f"(1.0f));
}

// Forward straight to E4M3 with one FP32 scale per 128 columns (sf = max(amax, 1e-4) / 448, q = e4m3(y / sf)): the products stay in FP32 until
// that one rounding, and all of it is FP32 arithmetic as its operations round (with an approximate exponential, reciprocal and quotient one code in a
// million was another). A lane owns 8 columns, 16 lanes a scale block; inter is a multiple of 8, a last block may be short. The issue slots
// bound it: 32768 x 2 x 2048 59.4 us with the approximate operations, 69.0 with these, 64.5 with the divisions shared out among a block's lanes.
template <int kRows>
__global__ void __launch_bounds__(256) dgb200_swiglu_cast_kernel(const SwigluParams p) {
    static_assert(kRows == 1 || kRows == 4, "lane l of a block divides for row l % kRows");
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
    float y[kRows][8], amax[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        float g[8], u[8];
        V::unpack(gate[r], g);
        V::unpack(up[r], u);
        if (p.clamp > 0.0f) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                g[i] = clamp_above(g[i], p.clamp);
                u[i] = clamp_both(u[i], p.clamp);
            }
        }
        amax[r] = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            swiglu_f32x2(g[i], g[i + 1], u[i], u[i + 1], y[r][i], y[r][i + 1]);
            amax[r] = fmaxf(amax[r], fmaxf(fabsf(y[r][i]), fabsf(y[r][i + 1])));
        }
#pragma unroll
        for (int off = 1; off < 16; off <<= 1) amax[r] = fmaxf(amax[r], __shfl_xor_sync(0xffffffffu, amax[r], off));
    }
    const int lane = static_cast<int>(threadIdx.x & 31), mine = lane % kRows;
    const float a = mine == 0 ? amax[0] : (mine == 1 ? amax[1 % kRows] : (mine == 2 ? amax[2 % kRows] : amax[3 % kRows]));
    const float my_sf = fmaxf(a, 1e-4f) / 448.0f;
    const float my_y = -1.0f / my_sf;
    // (of a short last block the storing lane itself may lie outside)
    if ((lane & 15) < kRows && col - (lane & 15) * 8 < p.inter && row0 + mine < rows) p.sf[(row0 + mine) * p.sf_stride + col / 128] = my_sf;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        const float sf = __shfl_sync(0xffffffffu, my_sf, (lane & 16) | r), minus_y = __shfl_sync(0xffffffffu, my_y, (lane & 16) | r);
        if (!inside || row0 + r >= rows) continue;
        float q[8];  // with the sign turned
        if (amax[r] == INFINITY) {
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] = y[r][i] / -sf;
        } else {
#pragma unroll
            for (int i = 0; i < 8; i += 2) negated_quotients(y[r][i], y[r][i + 1], sf, minus_y, q[i], q[i + 1]);
        }
        const __nv_fp8x4_e4m3 lo(make_float4(q[0], q[1], q[2], q[3]));
        const __nv_fp8x4_e4m3 hi(make_float4(q[4], q[5], q[6], q[7]));
        *reinterpret_cast<uint2*>(static_cast<unsigned char*>(p.out) + (row0 + r) * p.out_stride + col) =
            make_uint2(lo.__x ^ 0x80808080u, hi.__x ^ 0x80808080u);
    }
}

}  // namespace dgb
