// Gradients of the causal depthwise conv1d + bias + SiLU (m1_conv.cu).
//
//   pre[t]  = bias + sum_j w[j] x[t - K + 1 + j],   out[t] = silu(pre[t])
//   dpre[t] = dout[t] s (1 + pre (1 - s)),          s = sigmoid(pre[t])
//   dx[t]   = sum_j w[j] dpre[t + K - 1 - j]
//   dw[j]   = sum_{b,t} dpre[t] x[t - K + 1 + j],   dbias = sum_{b,t} dpre[t]
//
// Nothing of the forward is saved but x: pre is recomputed.  A warp walks a run
// of steps of one (batch, channel) row from its end to its start, 32 E steps at
// a time; a lane owns E consecutive steps.  x and dout arrive by cp.async in a
// ring of kStages iterations per warp (loads into registers did not stay ahead:
// the x before lane 0's steps is the next iteration's and is wanted at once);
// a lane reads its own steps and those before them from the ring, and gets the
// K - 1 dpre after its own from the lane above by shuffle (lane 31: kept from
// the last iteration).  So each value is loaded, and each dpre computed, once.
// dw and dbias are summed in registers, then over lanes, written as one partial
// per warp and added in a fixed order by a second kernel.
//
// Lanes sit on the 16-byte boundaries of memory, not on the row's start: a row
// of odd length begins `lead` elements past a boundary, and its steps are
// counted from that boundary (what comes before the row is masked).  So rows of
// any length take 16-byte accesses.
//
// Bound by HBM in fp32; in bf16 by the work per step (the shuffles, sigmoid and
// 3 K multiply-adds are the same for half the bytes): 8 x 1536 rows of
// 2048 steps, K = 4: 52 us in fp32 (302 MB, 5.8 TB/s, 89% of the measured copy
// rate), 44 us in bf16 (52%); 3 x 1000 rows of 1537 in bf16: 14 us.  x and dout have
// one type; bf16 x with fp32 dout is converted by the caller (144 us with the
// conversions, the same 8 x 1536 rows).
#include <algorithm>
#include <cstdint>

#include "common.cuh"
#include "train.h"

namespace b200scan {

namespace {

constexpr int kThreads = 128;

// Splits of a row into runs of whole 256-step pieces, so that few rows still
// fill the GPU: as many as keep to one wave of 32 warps per SM (2 splits of 3000
// rows, 1.3 waves, took 17.9 us where 1 takes 15.6).
constexpr int kPiece = 256;
// Steps of a lane: one 16-byte access, or enough for the K - 1 steps that a lane
// gets from its neighbour.
template <typename T, int K>
constexpr int lane_steps() { return sizeof(T) == 2 || K > 5 ? 8 : 4; }
// Pieces of a row, counted from the boundary at most 7 elements before it.
int64_t conv_pieces(int64_t len) { return (len + 7 + kPiece - 1) / kPiece; }
int64_t conv_splits(const ConvBwdParams& p) {
    const int64_t want = 148 * 32 / (p.batch * p.dim);
    return std::max<int64_t>(1, std::min(conv_pieces(p.len), want));
}

constexpr int kStages = 4;
// A warp's ring: kStages iterations of x and of dout.
template <typename T, int E>
struct Ring {
    T x[kStages][32 * E], g[kStages][32 * E];
};

// Starts the copy of a lane's E elements at `src`, of which the first `valid`
// are in the row; the rest become zero.
template <typename T, int E, bool VEC, bool FULL = false>
__device__ __forceinline__ void copy_run(T* dst, const T* __restrict__ src, int valid = E) {
    if constexpr (VEC && FULL) {
#pragma unroll
        for (int i = 0; i < E; i += 16 / sizeof(T))
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(
                             __cvta_generic_to_shared(dst + i))),
                         "l"(src + i)
                         : "memory");
    } else if constexpr (VEC) {
        constexpr int kV = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < E; i += kV) {
            const int bytes = max(0, min(valid - i, kV)) * static_cast<int>(sizeof(T));
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(static_cast<uint32_t>(
                             __cvta_generic_to_shared(dst + i))),
                         "l"(bytes ? src + i : src), "r"(bytes)
                         : "memory");
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) dst[e] = e < valid ? src[e] : from_f32<T>(0.f);
    }
}

// E elements of the ring as fp32.
template <typename T, int E>
__device__ __forceinline__ void read_run(const T* src, float* v) {
#pragma unroll
    for (int i = 0; i < E; i += 16 / sizeof(T)) {
        const uint4 a = *reinterpret_cast<const uint4*>(src + i);
        const uint32_t q[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (sizeof(T) == 4) {
                v[i + e] = __uint_as_float(q[e]);
            } else {
                v[i + 2 * e] = __uint_as_float(q[e] << 16);
                v[i + 2 * e + 1] = __uint_as_float(q[e] & 0xffff0000u);
            }
        }
    }
}

template <typename T, int E, bool VEC>
__device__ __forceinline__ void store_run(T* __restrict__ at, const float* o) {
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < E; i += 16 / sizeof(T)) {
            uint32_t q[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (sizeof(T) == 4) {
                    q[e] = __float_as_uint(o[i + e]);
                } else {
                    const __nv_bfloat162 v = __floats2bfloat162_rn(o[i + 2 * e], o[i + 2 * e + 1]);
                    q[e] = *reinterpret_cast<const uint32_t*>(&v);
                }
            }
            *reinterpret_cast<uint4*>(at + i) = make_uint4(q[0], q[1], q[2], q[3]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) at[e] = from_f32<T>(o[e]);
    }
}

// dpre from pre and dout; silu'(pre) = s (1 + pre (1 - s)).
__device__ __forceinline__ float dpre_of(float pre, float go) {
    const float s = rcp_approx(1.f + ex2_approx(-pre * kLog2e));
    return go * s * fmaf(pre, 1.f - s, 1.f);
}

template <typename T, int K, int kE, bool VEC>
__global__ void __launch_bounds__(kThreads) m1_conv_bwd_kernel(ConvBwdParams p, int64_t splits, int64_t pieces,
                                                               float* partial) {
    static_assert(K - 1 <= kE);
    constexpr int kRun = 32 * kE;  // steps of an iteration
    static_assert(kPiece % kRun == 0);
    constexpr unsigned kAll = 0xffffffffu;
    const int lane = threadIdx.x & 31;
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + threadIdx.x / 32;
    const int64_t rows = p.batch * p.dim;
    if (unit >= rows * splits) return;
    __shared__ __align__(16) Ring<T, kE> rings[kThreads / 32];
    Ring<T, kE>& ring = rings[threadIdx.x / 32];
    int64_t row, split, batch, d;
    divide(unit, splits, &row, &split);
    divide(row, p.dim, &batch, &d);
    const T* x = static_cast<const T*>(p.x) + row * p.len;
    const T* dout = static_cast<const T*>(p.dout) + row * p.len;
    T* dx = static_cast<T*>(p.dx) + row * p.len;
    // steps are counted from the boundary `lead` elements before the row (x,
    // dout and dx lie alike: the launcher's condition for VEC)
    const int lead = VEC ? static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T)) : 0;
    int64_t piece0, piece1, rest;
    divide(pieces * split, splits, &piece0, &rest);
    divide(pieces * (split + 1), splits, &piece1, &rest);
    const int64_t begin = piece0 * kPiece, end = min(piece1 * kPiece, lead + p.len);
    // sums[j]: dw[j], and dbias at K.  A lane adds up to kFlush iterations in `part`
    // first: a long row's sums keep the error of short ones (720001 steps: 1.6e-5 of
    // dbias without)
    constexpr int kFlush = 16;
    float w[K], sums[K + 1], part[K + 1];
#pragma unroll
    for (int j = 0; j <= K; ++j) sums[j] = part[j] = 0.f;
#pragma unroll
    for (int j = 0; j < K; ++j) w[j] = __ldg(p.w + d * K + j);
    const float b0 = p.bias ? __ldg(p.bias + d) : 0.f;
    // after[i]: dpre of the step i past the end of the current iteration.  At
    // first: the steps past this run, the next split's; lane i computes the i-th.
    float after[K > 1 ? K - 1 : 1];
    if (K > 1) {
        float v = 0.f;
        const int64_t t1 = end - lead + lane;
        if (lane < K - 1 && t1 < p.len) {
            float pre = b0;
#pragma unroll
            for (int j = 0; j < K; ++j) {
                const int64_t t = t1 - (K - 1) + j;
                if (t >= 0) pre = fmaf(w[j], to_f32(x[t]), pre);
            }
            v = dpre_of(pre, to_f32(dout[t1]));
        }
#pragma unroll
        for (int i = 0; i < K - 1; ++i) after[i] = __shfl_sync(kAll, v, i);
    }
    // Iterations start at multiples of kRun, which divides kPiece: only one that
    // holds the row's end is not full, and there dout, so dpre, is zero past it.
    const int iters = static_cast<int>((end - begin + kRun - 1) / kRun);
    if (iters > 0) {
        const int64_t s0 = begin + static_cast<int64_t>(iters - 1) * kRun + lane * kE;
        x += s0 - lead;
        dout += s0 - lead;
        dx += s0 - lead;
        // a lane's elements in the row: from `head` on in the row's first iteration (which
        // is iteration 0 of its first split only), up to `tail` in its last
        const bool has_first = begin == 0 && lead > 0;
        const int head = has_first ? max(0, lead - lane * kE) : 0;
        const int tail = static_cast<int>(max(static_cast<int64_t>(0), min(lead + p.len - s0, static_cast<int64_t>(kE))));
        const bool cut = lead + p.len - s0 + lane * kE < kRun;  // the last iteration holds the row's end
        // Iteration `it` (its first element `back` before the last iteration's).
        // Of the one below the run only the x before lane 0's steps are wanted;
        // before the row's start they are zero.
        auto start = [&](int it, int64_t back) {
            T* xd = ring.x[it & (kStages - 1)] + lane * kE;
            T* gd = ring.g[it & (kStages - 1)] + lane * kE;
            if (it > 0 && it < iters - 1) {
                copy_run<T, kE, VEC, true>(xd, x - back);
                copy_run<T, kE, VEC, true>(gd, dout - back);
            } else if (it >= 0) {
                const int valid = it == iters - 1 ? tail : kE;
                if (VEC && it == 0 && row == 0 && head > 0) {
                    // the boundary lies before the tensor: nothing is read there
#pragma unroll
                    for (int e = 0; e < kE; ++e) {
                        xd[e] = e >= head && e < valid ? x[e - back] : from_f32<T>(0.f);
                        gd[e] = e >= head && e < valid ? dout[e - back] : from_f32<T>(0.f);
                    }
                } else {
                    copy_run<T, kE, VEC>(xd, x - back, valid);
                    copy_run<T, kE, VEC>(gd, dout - back, valid);
                }
            } else if (it == -1 && lane == 31) {
                copy_run<T, kE, VEC>(xd, x - back, begin > 0 ? kE : 0);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int k = 0; k < kStages - 1; ++k) start(iters - 1 - k, static_cast<int64_t>(k) * kRun);
#pragma unroll 1
        for (int it = iters - 1; it >= 0; --it) {
            // this iteration's and the one below's copies are complete
            asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 3) : "memory");
            __syncwarp();
            // x over the kE steps before the lane's own, and these
            float win[2 * kE], go[kE];
            const T* xr = ring.x[it & (kStages - 1)] + lane * kE;
            read_run<T, kE>(lane ? xr - kE : ring.x[(it - 1) & (kStages - 1)] + 31 * kE, win);
            read_run<T, kE>(xr, win + kE);
            read_run<T, kE>(ring.g[it & (kStages - 1)] + lane * kE, go);
            if (it == 0 && has_first) {
#pragma unroll
                for (int e = 0; e < kE; ++e) {
                    if (e < head) win[kE + e] = go[e] = 0.f;
                    if (lane == 0 || lane * kE - kE + e < lead) win[e] = 0.f;
                }
            }
            __syncwarp();  // the stage that is filled next was read in the last iteration
            start(it - (kStages - 1), (kStages - 1) * kRun);
            float dpre[kE + K - 1];
#pragma unroll
            for (int e = 0; e < kE; ++e) {
                float pre = b0;
#pragma unroll
                for (int j = 0; j < K; ++j) pre = fmaf(w[j], win[kE - (K - 1) + e + j], pre);
                dpre[e] = dpre_of(pre, go[e]);
#pragma unroll
                for (int j = 0; j < K; ++j) part[j] = fmaf(dpre[e], win[kE - (K - 1) + e + j], part[j]);
                part[K] += dpre[e];
            }
            // dpre of the K - 1 steps after the lane's own
#pragma unroll
            for (int i = 0; i < K - 1; ++i) {
                const float next = __shfl_sync(kAll, dpre[i], lane + 1);  // lane 31: lane 0's
                dpre[kE + i] = lane < 31 ? next : after[i];
                after[i] = next;  // only lane 31's is used
            }
            float o[kE];
#pragma unroll
            for (int e = 0; e < kE; ++e) {
                o[e] = 0.f;
#pragma unroll
                for (int j = 0; j < K; ++j) o[e] = fmaf(w[j], dpre[e + K - 1 - j], o[e]);
            }
            if ((it == iters - 1 && cut) || (it == 0 && has_first)) {
                const int lo = it == 0 && has_first ? head : 0, hi = it == iters - 1 ? tail : kE;
#pragma unroll
                for (int e = 0; e < kE; ++e)
                    if (e >= lo && e < hi) dx[e] = from_f32<T>(o[e]);
            } else {
                store_run<T, kE, VEC>(dx, o);
            }
            x -= kRun;
            dout -= kRun;
            dx -= kRun;
            if (it % kFlush == 0) {
#pragma unroll
                for (int j = 0; j <= K; ++j) {
                    sums[j] += part[j];
                    part[j] = 0.f;
                }
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    griddep_launch_dependents();
#pragma unroll
    for (int j = 0; j <= K; ++j) {
        float v = sums[j];
#pragma unroll
        for (int m = 16; m; m >>= 1) v += __shfl_xor_sync(kAll, v, m);
        // partial[j][batch * splits + split][d]
        if (lane == 0) partial[(j * (p.batch * splits) + batch * splits + split) * p.dim + d] = v;
    }
}

// dw[d][j] and dbias[d]: the partials of channel d added in index order.
__global__ void m1_conv_bwd_reduce(const float* __restrict__ partial, int64_t parts, int64_t dim, int K,
                                   float* dw, float* dbias) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= dim * (K + 1)) return;
    int64_t j, d;
    divide(i, dim, &j, &d);
    griddep_wait();  // the partial sums
    float s = 0.f;
#pragma unroll 8
    for (int64_t k = 0; k < parts; ++k) s += partial[(j * parts + k) * dim + d];
    if (j < K) dw[d * K + j] = s;
    else if (dbias) dbias[d] = s;
}

template <typename T, int K>
void conv_bwd_start(const ConvBwdParams& p, int64_t splits, float* partial, cudaStream_t stream) {
    const int64_t units = p.batch * p.dim * splits;
    const unsigned g = static_cast<unsigned>((units + kThreads / 32 - 1) / (kThreads / 32));
    // 16-byte accesses where the three tensors lie alike on 16-byte boundaries
    const uintptr_t ax = reinterpret_cast<uintptr_t>(p.x), ag = reinterpret_cast<uintptr_t>(p.dout),
                    ao = reinterpret_cast<uintptr_t>(p.dx);
    const int64_t pieces = conv_pieces(p.len);
    if (((ax ^ ag) & 15u) == 0 && ((ax ^ ao) & 15u) == 0)
        m1_conv_bwd_kernel<T, K, lane_steps<T, K>(), true><<<g, kThreads, 0, stream>>>(p, splits, pieces, partial);
    else
        m1_conv_bwd_kernel<T, K, lane_steps<T, K>(), false><<<g, kThreads, 0, stream>>>(p, splits, pieces, partial);
}

template <typename T>
void conv_bwd_start_k(const ConvBwdParams& p, int64_t splits, float* partial, cudaStream_t stream) {
    switch (p.K) {
        case 1: conv_bwd_start<T, 1>(p, splits, partial, stream); break;
        case 2: conv_bwd_start<T, 2>(p, splits, partial, stream); break;
        case 3: conv_bwd_start<T, 3>(p, splits, partial, stream); break;
        case 4: conv_bwd_start<T, 4>(p, splits, partial, stream); break;
        case 5: conv_bwd_start<T, 5>(p, splits, partial, stream); break;
        case 6: conv_bwd_start<T, 6>(p, splits, partial, stream); break;
        case 7: conv_bwd_start<T, 7>(p, splits, partial, stream); break;
        default: conv_bwd_start<T, 8>(p, splits, partial, stream); break;
    }
}

}  // namespace

size_t m1_conv_bwd_workspace_bytes(const ConvBwdParams& p) {
    return static_cast<size_t>(p.K + 1) * p.batch * conv_splits(p) * p.dim * sizeof(float);
}

cudaError_t m1_conv_bwd_launch(const ConvBwdParams& p, void* workspace, cudaStream_t stream) {
    const int64_t splits = conv_splits(p);
    if (p.batch * p.dim * splits / (kThreads / 32) >= (int64_t(1) << 31) - 1) return cudaErrorInvalidValue;
    float* partial = static_cast<float*>(workspace);
    if (p.dtype == kF32) conv_bwd_start_k<float>(p, splits, partial, stream);
    else conv_bwd_start_k<__nv_bfloat16>(p, splits, partial, stream);
    note_launch();
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    const int64_t n = p.dim * (p.K + 1);
    e = launch_pdl(m1_conv_bwd_reduce, static_cast<unsigned>((n + 127) / 128), 128, stream, partial, p.batch * splits,
                   p.dim, p.K, p.dw, p.dbias);
    note_launch();
    return e;
}

}  // namespace b200scan
