// SwiGLU of the experts' rows, forward and backward, as operators of their own (the layers fuse the forward form into their
// gate/up GEMM). Rows are [gate | up]; with a clamp c the gate is min(gate, c) and up is clamped to [-c, c], and the
// gradient is zero where a clamp holds. Bound by HBM: every value is read and written once in 16-byte vectors, four rows a thread where
// there are many (32768 x 2 x 2048, call after call: forward 61.5 us, 6.5 TB/s, backward 100.5, 6.7; to FP8 71 us, with a clamp 81, where the issue
// slots are taken).
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

// 1 / (1 + e^-x) from the hardware's exponential and reciprocal. Relatively off by (2 + 1.16 |x|) 2^-23 of the exponential (as documented: it
// rounds its argument) where x is negative, and about 2^-22 more: 2^-16 at -87, against the 2^-9 of the BF16 rounding that follows. Below
// kFarGate the reciprocal would be a subnormal number, which the hardware's flushes to zero.
__device__ __forceinline__ float sigmoid_fast(float x) { return rcp_approx(1.0f + __expf(-x)); }

// Gates below kFarGate (e^87 lies under 2^126): 1 + e^g is one in FP32 and s = e^g = t^2 with t = e^(g / 2), a factor for each of the two
// others, so that nothing leaves the normal range that the product does not. They are rare, so the BF16 kernels look for them with a minimum over all of
// a thread's gates and mend what they gave behind the stores, in a function of its own. 32768 x 2 x 2048 at a low clock, forward and backward
// without any of it 62.7 and 102.7 us; as it is 63.6 and 104.7; with the function inlined 65 and 108.5; with every gate's root selected in line
// 71 and 119 (at a high clock as it is and without: 61.5 and 100.5 both).
constexpr float kFarGate = -87.0f;
__device__ __forceinline__ float far_product(float a, float b, float t) { return (a * t) * (b * t); }

// Minimum of the BF16 pairs in a vector; NaN is passed over.
__device__ __forceinline__ __nv_bfloat162 bf16x2_of(uint32_t w) {
    __nv_bfloat162 v;
    memcpy(&v, &w, 4);
    return v;
}
__device__ __forceinline__ __nv_bfloat162 lowest(const uint4& r) {
    return __hmin2(__hmin2(bf16x2_of(r.x), bf16x2_of(r.y)), __hmin2(bf16x2_of(r.z), bf16x2_of(r.w)));
}
__device__ __forceinline__ __nv_bfloat162 lowest(unsigned short r) { return bf16x2_of(r); }
__device__ __forceinline__ bool is_far(__nv_bfloat162 m) { return fminf(__low2float(m), __high2float(m)) < kFarGate; }

// The far gates among `columns` columns of some rows, once more.
__device__ __noinline__ void far_forward(const SwigluParams& p, int row0, int row_end, int col, int columns) {
#pragma unroll 1
    for (int row = row0; row < row_end; ++row)
#pragma unroll 1
        for (int c = col; c < col + columns; ++c) {
            const __nv_bfloat16* x = p.x + row * p.x_stride + c;
            const float g = __bfloat162float(x[0]), u = __bfloat162float(x[p.inter]);
            if (!(g < kFarGate)) continue;
            static_cast<__nv_bfloat16*>(p.out)[row * p.out_stride + c] =
                __float2bfloat16(far_product(g, p.clamp > 0.0f ? clamp_both(u, p.clamp) : u, __expf(0.5f * g)));
        }
}
__device__ __noinline__ void far_backward(const SwigluParams& p, int row0, int row_end, int col, int columns) {
#pragma unroll 1
    for (int row = row0; row < row_end; ++row)
#pragma unroll 1
        for (int c = col; c < col + columns; ++c) {
            const __nv_bfloat16* x = p.x + row * p.x_stride + c;
            const float g = __bfloat162float(x[0]), u = __bfloat162float(x[p.inter]), dy = __bfloat162float(p.dy[row * p.dy_stride + c]);
            if (!(g < kFarGate)) continue;
            const float t = __expf(0.5f * g);
            const bool held = p.clamp > 0.0f && fabsf(u) > p.clamp;
            __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out) + row * p.out_stride + c;
            out[0] = __float2bfloat16(far_product(dy, p.clamp > 0.0f ? clamp_both(u, p.clamp) : u, t) * (1.0f + g));
            out[p.inter] = __float2bfloat16(held ? 0.0f : far_product(dy, g, t));
        }
}

// One thread: kVec columns of kRows consecutive rows, so that 2 kRows loads (3 kRows backward) are in flight.
template <int kVec, int kRows>
__global__ void __launch_bounds__(256) dgb200_swiglu_kernel(const __grid_constant__ SwigluParams p) {
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
    __nv_bfloat162 low = bf16x2_of(0);
#pragma unroll
    for (int r = 0; r < kRows; ++r)
        if (row0 + r < rows) {
            low = __hmin2(low, lowest(gate[r]));
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
    if (is_far(low)) far_forward(p, row0, min(row0 + kRows, rows), col, kVec);
}

// d_gate = dy u s(g) (1 + g (1 - s(g))), d_up = dy g s(g); zero where the clamp holds.
template <int kVec, int kRows>
__global__ void __launch_bounds__(256) dgb200_swiglu_backward_kernel(const __grid_constant__ SwigluParams p) {
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
    __nv_bfloat162 low = bf16x2_of(0);
#pragma unroll
    for (int r = 0; r < kRows; ++r)
        if (row0 + r < rows) {
            low = __hmin2(low, lowest(gate[r]));
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
    if (is_far(low)) far_backward(p, row0, min(row0 + kRows, rows), col, kVec);
}

// 4 g u / (1 + e^-g) for two values, but for the factor as FP32 operations give it: the reciprocal is rounded correctly but for rare cases (one
// Newton step). The factor keeps the reciprocal of the largest finite e^-g, about 2^-128, out of the subnormal numbers, which the hardware's
// flushes to zero; where e^-g is infinite (g below -88.7) the step makes NaN of zero times infinity.
__device__ __forceinline__ void swiglu_times_4(float e0, float e1, float g0, float g1, float u0, float u1, float& y0, float& y1) {
    const float d0 = fmaf(e0, -0.25f, -0.25f), d1 = fmaf(e1, -0.25f, -0.25f);  // -(1 + e^-g) / 4
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
        "}\n" : "=f"(y0), "=f"(y1) : "f"(g0), "f"(g1), "f"(u0), "f"(u1), "f"(d0), "f"(d1), "f"(rcp_approx(-d0)), "f"(rcp_approx(-d1)), "f"(1.0f));
}

// Maximum that is NaN where one of the two is.
__device__ __forceinline__ float max_or_nan(float a, float b) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}

// Rows whose products hold NaN, an infinity or, before their factor of four is taken back, one too large for FP32, and those with far gates: the
// definition value by value, to the same bits where the quick way below serves. All lanes of the warp; rolled up, for it is rare.
__device__ __forceinline__ void swiglu_cast_special_row(const SwigluParams& p, int row, int col) {
    const __nv_bfloat16* x = p.x + row * p.x_stride + col;
    const int columns = min(p.inter - col, 8);  // of this lane; none or fewer than none in a short last block
    auto product = [&](int i) {
        float g = __bfloat162float(x[i]), u = __bfloat162float(x[p.inter + i]);
        if (p.clamp > 0.0f) {
            g = clamp_above(g, p.clamp);
            u = clamp_both(u, p.clamp);
        }
        if (g < kFarGate) return far_product(g, u, expf(0.5f * g));
        float y, same;
        swiglu_times_4(expf(-g), expf(-g), 0.25f * g, 0.25f * g, u, u, y, same);
        return y;
    };
    float amax = 0.0f;
#pragma unroll 1
    for (int i = 0; i < columns; ++i) amax = fmaxf(amax, fabsf(product(i)));
#pragma unroll 1
    for (int off = 1; off < 16; off <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
    const float sf = fmaxf(amax, 1e-4f) / 448.0f;
    if ((threadIdx.x & 15) == 0 && col < p.inter) p.sf[row * p.sf_stride + col / 128] = sf;
#pragma unroll 1
    for (int i = 0; i < columns; ++i)
        static_cast<unsigned char*>(p.out)[row * p.out_stride + col + i] = __nv_cvt_float_to_fp8(product(i) / sf, __NV_SATFINITE, __NV_E4M3);
}

// Forward straight to E4M3 with one FP32 scale per 128 columns (sf = max(amax, 1e-4) / 448, q = e4m3(y / sf)): the products stay in FP32 until
// that one rounding, and all of it is FP32 arithmetic as its operations round (with an approximate exponential, reciprocal and quotient one code in a
// million was another). A lane owns 8 columns, 16 lanes a scale block; inter is a multiple of 8, a last block may be short. The issue slots
// bound it: 32768 x 2 x 2048 59.4 us with the approximate operations, 69.0 with these, 64.5 with the divisions shared out among a block's lanes.
// Where the maximum of a block is no finite number, the warp's rows are done one by one instead: far gates and NaN pass through the maxima, an
// infinity may be the factor's. That costs 1 % where it is never taken (69.8 -> 71 us, with a clamp 80.0 -> 80.9); finding far gates by a minimum, 5 %.
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
    float y[kRows][8], amax[kRows];  // four times the products
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
            swiglu_times_4(expf(-g[i]), expf(-g[i + 1]), g[i], g[i + 1], u[i], u[i + 1], y[r][i], y[r][i + 1]);
            amax[r] = max_or_nan(amax[r], max_or_nan(fabsf(y[r][i]), fabsf(y[r][i + 1])));
        }
#pragma unroll
        for (int off = 1; off < 16; off <<= 1) amax[r] = max_or_nan(amax[r], __shfl_xor_sync(0xffffffffu, amax[r], off));
    }
    const int lane = static_cast<int>(threadIdx.x & 31), mine = lane % kRows;
    const float a = mine == 0 ? amax[0] : (mine == 1 ? amax[1 % kRows] : (mine == 2 ? amax[2 % kRows] : amax[3 % kRows]));
    if (__any_sync(0xffffffffu, !(a < INFINITY))) {
#pragma unroll 1
        for (int row = row0; row < min(row0 + kRows, rows); ++row) swiglu_cast_special_row(p, row, col);
        return;
    }
    const float my_sf = fmaxf(a, 4.0f * 1e-4f) / 448.0f;
    const float my_y = -1.0f / my_sf;
    // (of a short last block the storing lane itself may lie outside)
    if ((lane & 15) < kRows && col - (lane & 15) * 8 < p.inter && row0 + mine < rows) p.sf[(row0 + mine) * p.sf_stride + col / 128] = my_sf * 0.25f;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        const float sf = __shfl_sync(0xffffffffu, my_sf, (lane & 16) | r), minus_y = __shfl_sync(0xffffffffu, my_y, (lane & 16) | r);
        if (!inside || row0 + r >= rows) continue;
        float q[8];  // with the sign turned
#pragma unroll
        for (int i = 0; i < 8; i += 2) negated_quotients(y[r][i], y[r][i + 1], sf, minus_y, q[i], q[i + 1]);
        const __nv_fp8x4_e4m3 lo(make_float4(q[0], q[1], q[2], q[3]));
        const __nv_fp8x4_e4m3 hi(make_float4(q[4], q[5], q[6], q[7]));
        *reinterpret_cast<uint2*>(static_cast<unsigned char*>(p.out) + (row0 + r) * p.out_stride + col) =
            make_uint2(lo.__x ^ 0x80808080u, hi.__x ^ 0x80808080u);
    }
}

}  // namespace dgb
