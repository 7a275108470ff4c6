// RMS norm with the residual's addition: forward (output in the input's type
// or in e4m3 with one scale per row) and backward.
//
//   r    = residual + x                    (written in the residual stream's type)
//   rstd = 1 / sqrt(mean(r^2) + eps),  y = r rstd w
//   e4m3: scale = max(max|y| / 448, 2^-126) (1 for a row of zeros),  y8 = e4m3(y / scale)
//   dr   = rstd (dy w - xh mean(dy w xh)) + dres_out,   xh = r rstd
//   dw   = sum over rows of dy xh
//
// A group of WPR warps owns a row; a thread keeps its share of the row (at
// most kPer values) in registers, so every tensor is read or written once and
// the kernel is bound by HBM.  Sums are fp32: a thread adds at most kPer
// squares, the rest is a tree.  The backward kernel is persistent over rows,
// keeps the dw sums of its columns in registers and leaves one partial row
// per CTA; a second kernel adds the partials in a fixed order.
//
// Measured, 16384 rows of 768, bf16 on an fp32 residual: forward 23.9 us (151 MB,
// 6.3 TB/s), backward 29.2 + 4.9 us for dw's partials (201 MB, 6.9 TB/s with the
// writes that stay in L2).  Wide rows: 2048 of 8192 forward 34 us, backward 60 (31 and 41 at
// the copy rate), 1024 of 16384 39 and 72: 16 warps a row have no registers for the next
// row, and above 12288 columns the backward spills (232 to 460 bytes a thread).  A width
// or a start off 16 bytes is read element by element: 2048 of 8190 76 and 181 us.
// e4m3: 5003 rows of 2560 20 us (90 MB, 4.5 TB/s), 4 rows of 768 4.6 us.
#include <cuda_fp8.h>

#include <algorithm>
#include <cstdint>

#include "common.cuh"
#include "train.h"

namespace b200scan {

namespace {

constexpr int kPer = 32;  // values of a row one thread holds

// V consecutive elements at element offset `i` of a row.
template <typename T, int V>
__device__ __forceinline__ void load_v(const T* __restrict__ p, int64_t i, float* v) {
    if constexpr (V == 1) {
        v[0] = to_f32(p[i]);
    } else if constexpr (sizeof(T) == 4) {
        const float4 a = *reinterpret_cast<const float4*>(p + i);
        const float4 b = *reinterpret_cast<const float4*>(p + i + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        const uint4 a = *reinterpret_cast<const uint4*>(p + i);
        const uint32_t q[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[2 * e] = __uint_as_float(q[e] << 16);
            v[2 * e + 1] = __uint_as_float(q[e] & 0xffff0000u);
        }
    }
}

template <typename T, int V>
__device__ __forceinline__ void store_v(T* __restrict__ p, int64_t i, const float* v) {
    if constexpr (V == 1) {
        p[i] = from_f32<T>(v[0]);
    } else if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(p + i) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(p + i + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        uint32_t q[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
            q[e] = *reinterpret_cast<const uint32_t*>(&b);
        }
        *reinterpret_cast<uint4*>(p + i) = make_uint4(q[0], q[1], q[2], q[3]);
    }
}

// The norm's weight, fp32 or bf16.
template <int V>
__device__ __forceinline__ void load_w(const void* w, int dtype, int64_t i, float* v) {
    if (dtype == kF32) load_v<float, V>(static_cast<const float*>(w), i, v);
    else load_v<__nv_bfloat16, V>(static_cast<const __nv_bfloat16*>(w), i, v);
}

// Sum or maximum over the WPR warps of a row; every thread gets the result.
// NaN wins the maximum, so that a row with one shows it in its scale.
struct Sum {
    static __device__ __forceinline__ float of(float a, float b) { return a + b; }
};
struct Max {
    static __device__ __forceinline__ float of(float a, float b) { return a != a || a > b ? a : b; }
};
// `smem` (WPR floats) must not be used again before the next barrier.
template <typename Op, int WPR>
__device__ __forceinline__ float row_reduce(float v, float* smem) {
#pragma unroll
    for (int m = 16; m; m >>= 1) v = Op::of(v, __shfl_xor_sync(0xffffffffu, v, m));
    if constexpr (WPR > 1) {
        if ((threadIdx.x & 31) == 0) smem[threadIdx.x / 32] = v;
        __syncthreads();
        v = smem[0];
#pragma unroll
        for (int k = 1; k < WPR; ++k) v = Op::of(v, smem[k]);
    }
    return v;
}

// Threads of a CTA: one row of WPR warps, or kRowsSmall rows of one warp.
constexpr int kRowsSmall = 4;
template <int WPR>
constexpr int norm_threads() { return WPR == 1 ? 32 * kRowsSmall : 32 * WPR; }

template <typename TX, typename TR, int WPR, int V, int kN, bool Y8>
__global__ void __launch_bounds__(norm_threads<WPR>()) rms_norm_kernel(NormParams p) {
    constexpr int kT = 32 * WPR;
    __shared__ float red[2][WPR];
    const int64_t row = WPR == 1 ? static_cast<int64_t>(blockIdx.x) * kRowsSmall + threadIdx.x / 32 : blockIdx.x;
    const int tid = WPR == 1 ? threadIdx.x & 31 : threadIdx.x;
    if (row >= p.rows) return;  // whole warps of a one-warp row: no barrier follows
    const TX* x = static_cast<const TX*>(p.x) + row * p.x_stride;
    const TR* res = static_cast<const TR*>(p.residual) + row * p.res_stride;
    TR* ro = static_cast<TR*>(p.res_out) + row * p.dim;
    float r[kN][V];
    float ss = 0.f;
#pragma unroll
    for (int k = 0; k < kN; ++k) {
        const int64_t i = (static_cast<int64_t>(k) * kT + tid) * V;
        if (i < p.dim) {
            load_v<TX, V>(x, i, r[k]);
            if (p.residual) {
                float q[V];
                load_v<TR, V>(res, i, q);
#pragma unroll
                for (int e = 0; e < V; ++e) r[k][e] += q[e];
            }
            store_v<TR, V>(ro, i, r[k]);
#pragma unroll
            for (int e = 0; e < V; ++e) ss = fmaf(r[k][e], r[k][e], ss);
        }
    }
    ss = row_reduce<Sum, WPR>(ss, red[0]);
    const float rstd = 1.f / sqrtf(ss / static_cast<float>(p.dim) + p.eps);
    if (p.rstd && tid == 0) p.rstd[row] = rstd;
    float amax = 0.f;
#pragma unroll
    for (int k = 0; k < kN; ++k) {
        const int64_t i = (static_cast<int64_t>(k) * kT + tid) * V;
        if (i < p.dim) {
            float w[V];
            load_w<V>(p.w, p.w_dtype, i, w);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                r[k][e] = r[k][e] * rstd * w[e];
                if (Y8) amax = Max::of(amax, fabsf(r[k][e]));
            }
            if (!Y8) store_v<TX, V>(static_cast<TX*>(p.y) + row * p.dim, i, r[k]);
        }
    }
    if constexpr (Y8) {
        amax = row_reduce<Max, WPR>(amax, red[1]);
        // not below the least normal number, so that 1 / scale is finite (NaN stays)
        float scale = amax / 448.f;
        if (scale < 1.17549435e-38f) scale = amax == 0.f ? 1.f : 1.17549435e-38f;
        if (tid == 0) p.scale[row] = scale;
        // A product with 1 / scale (two more roundings of fp32 before the one to 8
        // bits): where y / scale lies within 1e-7 of the middle between two 8-bit
        // values the other one may be written, as near as the first.  5003 rows of
        // 2560: 19.9 us, with the quotient 24.0.
        const float inv = 1.f / scale;
        __nv_fp8_storage_t* y = static_cast<__nv_fp8_storage_t*>(p.y) + row * p.dim;
#pragma unroll
        for (int k = 0; k < kN; ++k) {
            const int64_t i = (static_cast<int64_t>(k) * kT + tid) * V;
            if (i < p.dim) {
                if constexpr (V == 1) {
                    y[i] = __nv_cvt_float_to_fp8(r[k][0] * inv, __NV_SATFINITE, __NV_E4M3);
                } else {
                    uint32_t q[V / 2];
#pragma unroll
                    for (int e = 0; e < V / 2; ++e)
                        q[e] = __nv_cvt_float2_to_fp8x2(make_float2(r[k][2 * e] * inv, r[k][2 * e + 1] * inv),
                                                        __NV_SATFINITE, __NV_E4M3);
                    *reinterpret_cast<uint2*>(y + i) = make_uint2(q[0] | q[1] << 16, q[2] | q[3] << 16);
                }
            }
        }
    }
}

bool aligned16(const void* a) { return (reinterpret_cast<uintptr_t>(a) & 15u) == 0; }

template <typename TX, typename TR, int WPR, int V, bool Y8>
void norm_width(const NormParams& p, cudaStream_t stream) {
    const unsigned g = static_cast<unsigned>(WPR == 1 ? (p.rows + kRowsSmall - 1) / kRowsSmall : p.rows);
    // runs a thread needs: fewer registers for narrower rows
    const int64_t runs = (p.dim + 32 * WPR * V - 1) / (32 * WPR * V);
    constexpr int kMax = kPer / V;
    if (runs <= kMax / 4) rms_norm_kernel<TX, TR, WPR, V, kMax / 4, Y8><<<g, norm_threads<WPR>(), 0, stream>>>(p);
    else if (runs <= kMax / 2) rms_norm_kernel<TX, TR, WPR, V, kMax / 2, Y8><<<g, norm_threads<WPR>(), 0, stream>>>(p);
    else if (runs <= kMax * 3 / 4) rms_norm_kernel<TX, TR, WPR, V, kMax * 3 / 4, Y8><<<g, norm_threads<WPR>(), 0, stream>>>(p);
    else rms_norm_kernel<TX, TR, WPR, V, kMax, Y8><<<g, norm_threads<WPR>(), 0, stream>>>(p);
}

template <typename TX, typename TR, int V>
cudaError_t norm_start(const NormParams& p, cudaStream_t stream) {
    // Warps per row by the row's width: a thread holds at most kPer values.  With
    // fewer rows than would give each SM one, four warps share a narrow row too:
    // the call's latency is then a row's (4 rows of 768: 4.7 us against 5.6).
    const bool few = p.rows <= 148 && p.dim > 32 * V;
    const int wpr = p.dim <= 32 * kPer && !few ? 1 : p.dim <= 4 * 32 * kPer ? 4 : 16;
    if (p.y8) {
        if (wpr == 1) norm_width<TX, TR, 1, V, true>(p, stream);
        else if (wpr == 4) norm_width<TX, TR, 4, V, true>(p, stream);
        else norm_width<TX, TR, 16, V, true>(p, stream);
    } else {
        if (wpr == 1) norm_width<TX, TR, 1, V, false>(p, stream);
        else if (wpr == 4) norm_width<TX, TR, 4, V, false>(p, stream);
        else norm_width<TX, TR, 16, V, false>(p, stream);
    }
    note_launch();
    return cudaGetLastError();
}

// V elements as they lie in memory.
template <typename T, int V>
struct Raw {
    static constexpr int kWords = V * sizeof(T) >= 4 ? V * sizeof(T) / 4 : 1;
    uint32_t w[kWords];
    __device__ __forceinline__ void load(const T* at) {
        if constexpr (V == 1) {
            if constexpr (sizeof(T) == 4) w[0] = __float_as_uint(*at);
            else w[0] = static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(at)) << 16;
        } else {
#pragma unroll
            for (int j = 0; j < kWords; j += 4) {
                const uint4 v = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(at) + j);
                w[j] = v.x; w[j + 1] = v.y; w[j + 2] = v.z; w[j + 3] = v.w;
            }
        }
    }
    __device__ __forceinline__ void get(float* v) const {
        if constexpr (V == 1 || sizeof(T) == 4) {
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = __uint_as_float(w[e]);
        } else {
#pragma unroll
            for (int j = 0; j < kWords; ++j) {
                v[2 * j] = __uint_as_float(w[j] << 16);
                v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
            }
        }
    }
};

// ---- backward --------------------------------------------------------------
// CTAs per SM: registers for a row (`values` of it a thread), the next row as it
// lies in memory and dw; a 16-bit residual stream leaves room for three.
constexpr int bwd_ctas_sm(int wpr, int res_bytes, int values) {
    return wpr == 16 ? 1 : res_bytes == 2 && values <= 24 ? 3 : 2;
}

// A thread's values of a row: N runs of V elements.  All loads of a row (dy, r,
// dres_out) are issued together, a row ahead where registers allow (16384 rows
// of 768, bf16 on fp32: 29.3 us with 8 warps a SM, without 34.2 us with 16; bf16 on
// bf16: 18.0 and 25.1).  Rows of 16 warps have no registers for the next row, and
// read dres_out last.
template <typename TY, typename TR, int WPR, int V, int N>
__global__ void __launch_bounds__(norm_threads<WPR>(), bwd_ctas_sm(WPR, sizeof(TR), N * V))
    rms_norm_bwd_kernel(NormBwdParams p, float* partial) {
    constexpr int kT = 32 * WPR;
    constexpr int kRows = WPR == 1 ? kRowsSmall : 1;
    __shared__ float red[2][WPR];
    int turn = 0;  // the buffer of a row: a warp may still read the last row's
    const int slot = WPR == 1 ? threadIdx.x / 32 : 0;
    const int tid = WPR == 1 ? threadIdx.x & 31 : threadIdx.x;
    float dw[N][V];
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) dw[k][e] = 0.f;
    constexpr bool kAhead = WPR < 16;
    const int64_t row_step = static_cast<int64_t>(gridDim.x) * kRows;
    Raw<TY, V> ndy[N];
    Raw<TR, V> nres[N], ndro[N];
    float nrstd = 0.f;
    auto fetch = [&](int64_t row) {
        nrstd = p.rstd[row];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int64_t i = (static_cast<int64_t>(k) * kT + tid) * V;
            if (i < p.dim) {
                ndy[k].load(static_cast<const TY*>(p.dy) + row * p.dim + i);
                nres[k].load(static_cast<const TR*>(p.res) + row * p.dim + i);
                if (kAhead && p.dres_out) ndro[k].load(static_cast<const TR*>(p.dres_out) + row * p.dim + i);
            }
        }
    };
    int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + slot;
    if (kAhead && row < p.rows) fetch(row);
    for (; row < p.rows; row += row_step) {
        if (!kAhead) fetch(row);
        const float rstd = nrstd;
        float xh[N][V], g[N][V], q[kAhead ? N : 1][V], c = 0.f;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            ndy[k].get(g[k]);
            nres[k].get(xh[k]);
            if constexpr (kAhead) ndro[k].get(q[k]);
        }
        if (kAhead && row + row_step < p.rows) fetch(row + row_step);
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int64_t i = (static_cast<int64_t>(k) * kT + tid) * V;
            if (i < p.dim) {
                float w[V];
                load_w<V>(p.w, p.w_dtype, i, w);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    xh[k][e] *= rstd;
                    dw[k][e] = fmaf(g[k][e], xh[k][e], dw[k][e]);
                    g[k][e] *= w[e];
                    c = fmaf(g[k][e], xh[k][e], c);
                }
            }
        }
        c = row_reduce<Sum, WPR>(c, red[turn]) / static_cast<float>(p.dim);
        turn ^= 1;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int64_t i = (static_cast<int64_t>(k) * kT + tid) * V;
            if (i < p.dim) {
                float* qk = q[kAhead ? k : 0];
                if (!kAhead && p.dres_out) load_v<TR, V>(static_cast<const TR*>(p.dres_out) + row * p.dim, i, qk);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    g[k][e] = rstd * fmaf(-xh[k][e], c, g[k][e]);
                    if (p.dres_out) g[k][e] += qk[e];
                }
                store_v<TY, V>(static_cast<TY*>(p.dx) + row * p.dim, i, g[k]);
                if (p.dres) store_v<TR, V>(static_cast<TR*>(p.dres) + row * p.dim, i, g[k]);
            }
        }
    }
    griddep_launch_dependents();
    // one partial row per CTA: the sums of its kRows warps, added in order
    float* out = partial + static_cast<int64_t>(blockIdx.x) * p.dim;
    if constexpr (kRows == 1) {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int64_t i = (static_cast<int64_t>(k) * kT + tid) * V;
            if (i < p.dim) store_v<float, V>(out, i, dw[k]);
        }
    } else {
        __shared__ float sums[kRows][32 * N * V];
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) sums[slot][(k * kT + tid) * V + e] = dw[k][e];
        __syncthreads();
        for (int i = threadIdx.x; i < p.dim; i += kRows * 32) {
            float v = sums[0][i];
#pragma unroll
            for (int k = 1; k < kRows; ++k) v += sums[k][i];
            out[i] = v;
        }
    }
}

// dw[c] = sum of the partial rows: a CTA takes 32 columns, each of its 32 warps
// every 32nd row; the 32 sums are added as a tree.
__global__ void __launch_bounds__(1024) rms_norm_dw_kernel(const float* __restrict__ partial, int64_t parts,
                                                           int64_t dim, float* dw) {
    __shared__ float s[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    float v = 0.f;
    griddep_wait();  // the partial rows
    if (c < dim) {
#pragma unroll 4
        for (int64_t k = warp; k < parts; k += 32) v += partial[k * dim + c];
    }
    s[warp][lane] = v;
    __syncthreads();
    v = s[lane][warp];  // row slice `lane` of column `warp`
#pragma unroll
    for (int m = 16; m; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    const int64_t col = static_cast<int64_t>(blockIdx.x) * 32 + warp;
    if (lane == 0 && col < dim) dw[col] = v;
}

int bwd_wpr(int64_t dim) { return dim <= 32 * kPer ? 1 : dim <= 4 * 32 * kPer ? 4 : 16; }

// CTAs of the persistent backward kernel with `per_sm` on each SM.
int64_t bwd_ctas(const NormBwdParams& p, int per_sm) {
    const int64_t need = bwd_wpr(p.dim) == 1 ? (p.rows + kRowsSmall - 1) / kRowsSmall : p.rows;
    return std::min<int64_t>(need, 148 * per_sm);
}

template <typename TY, typename TR, int WPR, int V, int N>
int64_t bwd_run(const NormBwdParams& p, float* partial, cudaStream_t stream) {
    const int64_t ctas = bwd_ctas(p, bwd_ctas_sm(WPR, sizeof(TR), N * V));
    rms_norm_bwd_kernel<TY, TR, WPR, V, N>
        <<<static_cast<unsigned>(ctas), norm_threads<WPR>(), 0, stream>>>(p, partial);
    return ctas;
}

template <typename TY, typename TR, int WPR, int V>
int64_t bwd_width(const NormBwdParams& p, float* partial, cudaStream_t stream) {
    // runs a thread needs: fewer registers for narrower rows
    const int64_t runs = (p.dim + 32 * WPR * V - 1) / (32 * WPR * V);
    constexpr int kMax = kPer / V;
    if (runs <= kMax / 4) return bwd_run<TY, TR, WPR, V, kMax / 4>(p, partial, stream);
    if (runs <= kMax / 2) return bwd_run<TY, TR, WPR, V, kMax / 2>(p, partial, stream);
    if (runs <= kMax * 3 / 4) return bwd_run<TY, TR, WPR, V, kMax * 3 / 4>(p, partial, stream);
    return bwd_run<TY, TR, WPR, V, kMax>(p, partial, stream);
}

template <typename TY, typename TR, int V>
cudaError_t bwd_start(const NormBwdParams& p, float* partial, cudaStream_t stream) {
    const int wpr = bwd_wpr(p.dim);
    const int64_t ctas = wpr == 1   ? bwd_width<TY, TR, 1, V>(p, partial, stream)
                         : wpr == 4 ? bwd_width<TY, TR, 4, V>(p, partial, stream)
                                    : bwd_width<TY, TR, 16, V>(p, partial, stream);
    note_launch();
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    e = launch_pdl(rms_norm_dw_kernel, static_cast<unsigned>((p.dim + 31) / 32), 1024, stream, partial, ctas, p.dim,
                   p.dw);
    note_launch();
    return e;
}

}  // namespace

cudaError_t rms_norm_launch(const NormParams& p, cudaStream_t stream) {
    if (p.rows >= (int64_t(1) << 31) - 1) return cudaErrorInvalidValue;
    const bool vec = p.dim % 8 == 0 && p.x_stride % 8 == 0 && p.res_stride % 8 == 0 && aligned16(p.x) &&
                     aligned16(p.residual) && aligned16(p.w) && aligned16(p.y) && aligned16(p.res_out);
    if (p.x_dtype == kF32)
        return vec ? norm_start<float, float, 8>(p, stream) : norm_start<float, float, 1>(p, stream);
    if (p.res_dtype == kF32)
        return vec ? norm_start<__nv_bfloat16, float, 8>(p, stream) : norm_start<__nv_bfloat16, float, 1>(p, stream);
    return vec ? norm_start<__nv_bfloat16, __nv_bfloat16, 8>(p, stream)
               : norm_start<__nv_bfloat16, __nv_bfloat16, 1>(p, stream);
}

size_t rms_norm_bwd_workspace_bytes(const NormBwdParams& p) {
    // of the most CTAs any type takes
    return static_cast<size_t>(bwd_ctas(p, 3)) * p.dim * sizeof(float);
}

cudaError_t rms_norm_bwd_launch(const NormBwdParams& p, void* workspace, cudaStream_t stream) {
    float* partial = static_cast<float*>(workspace);
    const bool vec = p.dim % 8 == 0 && aligned16(p.dy) && aligned16(p.res) && aligned16(p.w) &&
                     aligned16(p.dres_out) && aligned16(p.dx) && aligned16(p.dres) && aligned16(partial);
    if (p.dy_dtype == kF32)
        return vec ? bwd_start<float, float, 8>(p, partial, stream) : bwd_start<float, float, 1>(p, partial, stream);
    if (p.res_dtype == kF32)
        return vec ? bwd_start<__nv_bfloat16, float, 8>(p, partial, stream)
                   : bwd_start<__nv_bfloat16, float, 1>(p, partial, stream);
    return vec ? bwd_start<__nv_bfloat16, __nv_bfloat16, 8>(p, partial, stream)
               : bwd_start<__nv_bfloat16, __nv_bfloat16, 1>(p, partial, stream);
}

}  // namespace b200scan
