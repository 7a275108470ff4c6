// Gradients of the Mamba-1 selective scan.
//
// Forward, per (batch, channel) row and state n (the scan kernels' recurrence):
//   x = delta + bias;  dt = softplus(x) or x;  a = exp(dt A_n)
//   h_t = a_t h_{t-1} + dt u B_n;  y = sum_n C_n h + D u;  out = y silu(z)
// Given dout = dL/dout (and dlast = dL/dh_last), with s = sigmoid(z):
//   dy = dout z s;  dz = dout s (1 + z (1 - s)) y
//   g_t = dy_t C_n + a_{t+1} g_{t+1}                 (g = dL/dh; dlast enters last)
//   dC_n = sum_d dy h;  dB_n = sum_d g dt u
//   SB = sum_n g B_n;   SA = sum_n A_n g (a h_{t-1})
//   du = D dy + dt SB;  ddelta = (u SB + SA) dt/dx
//   dA_n = sum_{b,t} dt g (a h_{t-1});  dD = sum dy u;  dbias = sum ddelta;  dh0 = a_1 g_1
// Nothing of the forward is saved but its inputs.
//
// Passes: (1) a forward sweep leaves the state at the start of every block of
// kT steps; (2) with more than one time segment per row, a carry kernel turns
// segment aggregates into incoming states and gradients; (3) the main kernel
// walks the blocks backwards: it rescans a block from its saved state keeping
// a and a h_{t-1} of its kT steps in registers, then runs g back through them;
// (4) partial sums of dB, dC (over channels) and dA, dD, dbias (over batch and
// segments) are added in a fixed order.
//
// A warp owns 16 rows of one (batch, group); four lanes share a row, lane q
// holding states 4q..4q+3, and each lane works on two rows at once, so that a
// step's B and C, read from shared memory, serve eight (row, state) pairs: the
// loads' return path (4 bytes a lane and cycle) is what binds this kernel with
// one row a lane (11 of its cycles per warp-wide pair, 7 with two rows).
// Sums across lanes are butterflies in which a lane's slots are permuted by
// its own position, so the value to send and the one to keep sit in fixed
// registers and need no selects: state slot s of a lane in row r holds state
// 4q + (s ^ (r & 3)) (sums over channels: dB, dC), and row slot k of lane q
// holds row r + 8 (k ^ (q >> 1)) (sums over states: y, SB, SA).
// More than 16 states run as blocks of 16, one after the other.
//
// Measured at 8 x 1536 rows of 2048 steps, 16 states, fp32: 760 us (sweep 222,
// carries 10, main 530, sums 20 when timed apart).  Floors: 709 MB at 6.55 TB/s 108
// us, 9.9 GFLOP at the fp32 pipes' 72 TFLOP/s 137 us.  The passes' own decays, two
// per (row, step, state) and, in rows cut into segments, one per block of four
// steps, take 201 us at 16 exponentials a cycle and SM.  What binds it is latency: the main
// kernel issues on 53% of cycles with 3 warps a scheduler (168 registers: a and
// a h_{t-1} of eight pairs over four steps are 64 of them), its shared-memory
// path is 61% busy, FP32 pipes 42%, MUFU 31%, HBM 25%.  Of its time the
// elementwise part of a tile takes about 56 us, the gradients' stores 50, the
// states' correction in split rows 39, the row butterflies 20.
#include <algorithm>
#include <cstdint>
#include <initializer_list>
#include <type_traits>

#include "common.cuh"
#include "train.h"

namespace b200scan {

namespace {

constexpr int kT = 4;        // steps of a block: a and a h_{t-1} live in registers
constexpr int kTile = 16;    // steps staged at a time
constexpr int kTileBlocks = kTile / kT;
constexpr int kWarps = 4;
constexpr int kRowsW = 16;   // rows of a warp
constexpr int kRowsC = kWarps * kRowsW;    // rows of a CTA: a group's channels are padded to it
constexpr int kThreads = kWarps * 32;
constexpr int kStates = 16;
constexpr int kRowPitch = kTile + 4;       // floats between rows of a staged tensor
constexpr int kUpper = 16;                 // further floats before rows 8..15: other banks than rows 0..7
constexpr int kWarpRows = kRowsW * kRowPitch + kUpper;
constexpr int kBcPitch = 4 * kStates + 4;  // floats between steps of a staged B or C
constexpr int kSegTiles = 8;               // most tiles of a time segment
constexpr int kCtasSm = 3;                 // resident CTAs of the main kernel per SM

// How a launch cuts the problem.
struct Plan {
    int64_t per;       // channels of a group
    int64_t rblocks;   // CTAs covering a group's channels
    int64_t units;     // batch * groups * rblocks
    int64_t tiles;     // ceil(len / kTile)
    int64_t segs;      // time segments
    int64_t seg_tiles; // tiles of a segment
    int64_t blocks;    // ceil(len / kT) rounded up to whole tiles
    int width, gwidth; // bytes of one asynchronous copy of the activations, of dout (0: element loads)
    int width_out;     // 16: gradients of four steps are stored at once
};

// Widest copy that fits every tile of rows `len` elements apart at `ptrs`: tiles
// start at multiples of kTile steps (from the end, walked in reverse).
int copy_width(int64_t len, int size, std::initializer_list<const void*> ptrs) {
    uintptr_t bits = static_cast<uintptr_t>(len) * size;
    for (const void* v : ptrs) bits |= reinterpret_cast<uintptr_t>(v);
    return bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 0;
}

Plan make_plan(const M1BwdParams& p) {
    Plan q;
    q.width = copy_width(p.len, p.dtype == kF32 ? 4 : 2, {p.u, p.delta, p.z});
    q.gwidth = copy_width(p.len, p.dout_dtype == kF32 ? 4 : 2, {p.dout});
    q.width_out = copy_width(p.len, 4, {p.du, p.ddelta, p.dz});
    q.per = p.dim / p.groups;
    q.rblocks = (q.per + kRowsC - 1) / kRowsC;
    q.units = p.batch * p.groups * q.rblocks;
    q.tiles = (p.len + kTile - 1) / kTile;
    // Segments: of at most 128 steps, since the roundings of the decays add up along
    // a recurrence, and a carry between segments takes one decay of summed dt instead
    // (error of dA, 8 x 1536 rows of 2048 steps: 1.07e-6 in 10 segments, 9.3e-7 in 16;
    // with a scan by doubling spans in fp32 7.3e-7.  1 x 1536 rows of 32768: 1.20e-6 in
    // 128, 9.9e-7 in 256; 1.02e-6).  Among the numbers that give the SMs 1, 2, .. 36
    // CTAs each, the one with the least estimated time: a tile takes 7, 9 or 12 units
    // with 1, 2 or 3 CTAs on its SM; full waves run at 3, the rest at what is left; a
    // CTA's start-up and the carries count as one and a half tiles; CTAs that all
    // start together stay in step and get in each other's way (a tenth, over the
    // number of waves).  Measured, the same rows: 16 segments 760 us, 13: 746, 32:
    // 794; 256 segments 1453 us, 128: 1421, 410: 1504.  (The units were fitted to 16
    // states in fp32 and serve every state count and type.)
    q.seg_tiles = q.tiles;
    if (const int forced = kernel_override(kKnobM1Segments)) {
        q.seg_tiles = (q.tiles + forced - 1) / forced;
    } else {
        constexpr int64_t kSms = 148, kSlots = kSms * kCtasSm;
        constexpr double kTime[kCtasSm + 1] = {0.0, 7.1, 9.0, 11.8};
        const int64_t fewest = (q.tiles + kSegTiles - 1) / kSegTiles;
        double best = 0.0;
        for (int64_t m = 1; m <= 36; ++m) {
            const int64_t segs = std::min(q.tiles, std::max(fewest, m * kSms / q.units));
            const int64_t st = (q.tiles + segs - 1) / segs, n = (q.tiles + st - 1) / st;
            const int64_t waves = q.units * n / kSlots, rest = q.units * n % kSlots;
            const double cost = (st + 1.5) * (waves * kTime[kCtasSm] + kTime[(rest + kSms - 1) / kSms]) *
                                (1.0 + 0.1 / (waves + 1));
            if (m == 1 || cost < best) {
                best = cost;
                q.seg_tiles = st;
            }
            if (segs == q.tiles) break;
        }
    }
    q.segs = (q.tiles + q.seg_tiles - 1) / q.seg_tiles;
    q.blocks = q.tiles * kTileBlocks;
    return q;
}

// Workspace, in floats; every array starts on a 256-byte boundary.  "Warps" are
// units * kWarps groups of kRowsW rows; per-lane values are float4 over the
// four state slots.
struct Ws {
    float4* ckpt;    // [warps][blocks][2][32]: state at block starts, per row slot
    float* sdt;      // [warps][blocks][16]: dt log2(e) summed from the segment start
    float4* hend;    // [segs][warps][2][32]: end state from zero, then incoming state
    float4* gend;    // [segs][warps][2][32]: outgoing gradient from zero, then incoming
    float* stot;     // [segs][warps][16]: dt log2(e) summed over a segment
    float* dbp;      // [units][16][tiles * kTile] partial dB
    float* dcp;      // [units][16][tiles * kTile]
    float4* dap;     // [segs][warps][2][32] partial dA
    float* ddp;      // [segs][warps][16] partial dD
    float* dbiasp;   // [segs][warps][16]
    float* acc;      // [3][batch * dim * len] y, SB, SA over state blocks (state > 16)
    size_t floats;
};

Ws make_ws(const M1BwdParams& p, const Plan& q, void* base) {
    Ws w;
    float* f = static_cast<float*>(base);
    size_t n = 0;
    auto take = [&](size_t floats) {
        float* at = f + n;
        n += (floats + 63) / 64 * 64;
        return at;
    };
    const size_t uw = static_cast<size_t>(q.units) * kWarps;
    const bool split = q.segs > 1;
    w.ckpt = reinterpret_cast<float4*>(take(uw * q.blocks * 256));
    w.sdt = take(split ? uw * q.blocks * kRowsW : 0);
    w.hend = reinterpret_cast<float4*>(take(split ? q.segs * uw * 256 : 0));
    w.gend = reinterpret_cast<float4*>(take(split ? q.segs * uw * 256 : 0));
    w.stot = take(split ? q.segs * uw * kRowsW : 0);
    w.dbp = take(static_cast<size_t>(q.units) * kStates * q.tiles * kTile);
    w.dcp = take(static_cast<size_t>(q.units) * kStates * q.tiles * kTile);
    w.dap = reinterpret_cast<float4*>(take(q.segs * uw * 256));
    w.ddp = take(q.segs * uw * kRowsW);
    w.dbiasp = take(q.segs * uw * kRowsW);
    w.acc = take(p.state > kStates ? 3 * static_cast<size_t>(p.batch) * p.dim * p.len : 0);
    w.floats = n;
    return w;
}

struct Lane {
    int lane, q, r;        // state quarter, row (of 8) within the warp
    int64_t unit, seg, b, g;
    int64_t warp_id;       // number of the warp's 16 rows
    int64_t g0, d0;        // first channel of the warp, in its group and in all
    int rows;              // of the warp's 16 that exist
    __device__ __forceinline__ int row(int k) const { return r + 8 * (k ^ (q >> 1)); }
    __device__ __forceinline__ bool live(int k) const { return row(k) < rows; }
};

__device__ __forceinline__ Lane where(const M1BwdParams& p, const Plan& q) {
    Lane l;
    l.lane = threadIdx.x & 31;
    l.q = l.lane & 3;
    l.r = l.lane >> 2;
    int64_t bg, rb;
    divide(blockIdx.x, q.units, &l.seg, &l.unit);
    divide(l.unit, q.rblocks, &bg, &rb);
    divide(bg, p.groups, &l.b, &l.g);
    l.warp_id = l.unit * kWarps + threadIdx.x / 32;
    l.g0 = rb * kRowsC + (threadIdx.x / 32) * kRowsW;
    l.d0 = l.g * q.per + l.g0;
    l.rows = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(kRowsW), q.per - l.g0)));
    return l;
}

// Offset of a row within a warp's staged tensor.
__device__ __forceinline__ int row_at(int row) { return row * kRowPitch + (row >= 8 ? kUpper : 0); }

// State of slot s of a lane, within a block of 16.
__device__ __forceinline__ int slot_state(const Lane& l, int s) { return 4 * l.q + (s ^ (l.r & 3)); }

__device__ __forceinline__ int64_t step_of(const M1BwdParams& p, int64_t t) {
    return p.reverse ? p.len - 1 - t : t;
}

// dt and its derivative by x, with y = e^-|x| <= 1:
//   softplus(x) = max(x, 0) + log1p(y),  log1p(y) = 2 atanh(v), v = y / (2 + y) <= 1/3,
// the odd series of atanh to v^13 (truncation below 3e-8 of the result), and
// sigmoid(x) = 1 / (1 + y) or y / (1 + y).  dt enters every decay's exponent,
// so it is kept to a few roundings (lg2.approx loses 3e-6 near dt = 0.1).
template <bool SOFTPLUS>
__device__ __forceinline__ void dt_of(float x, float* dt, float* slope) {
    if constexpr (SOFTPLUS) {
        const float y = ex2_approx(-fabsf(x) * kLog2e);
        const float v = y * rcp_approx(2.f + y), q = v * v;
        float f = fmaf(q, 1.f / 13.f, 1.f / 11.f);
        f = fmaf(q, f, 1.f / 9.f);
        f = fmaf(q, f, 1.f / 7.f);
        f = fmaf(q, f, 1.f / 5.f);
        f = fmaf(q, f, 1.f / 3.f);
        const float l = fmaf(v * q, f, v);
        const float r = rcp_approx(1.f + y);
        const bool linear = x > 20.f;  // the scan's threshold: softplus(x) = x
        *dt = linear ? x : fmaf(2.f, l, fmaxf(x, 0.f));
        *slope = linear ? 1.f : x >= 0.f ? r : y * r;
    } else {
        *dt = x;
        *slope = 1.f;
    }
}

// Calls f with the call's flags (softplus, z given) as compile-time values, so
// that the elementwise loops hold no branches.
template <typename F>
__device__ __forceinline__ void with_flags(const M1BwdParams& p, F f) {
    using Yes = std::true_type;
    using No = std::false_type;
    if (p.delta_softplus) {
        if (p.z) f(Yes{}, Yes{});
        else f(Yes{}, No{});
    } else {
        if (p.z) f(No{}, Yes{});
        else f(No{}, No{});
    }
}

// B and C of one tile: a thread takes four states of one step, threads 0..63 B,
// 64..127 C.  They are loaded a tile ahead and then stored as four permuted
// copies per step: copy c holds state 4q + j at 4q + (j ^ c), which is the slot
// order of lanes with (row & 3) = c.
template <typename T>
__device__ __forceinline__ void load_bc(const M1BwdParams& p, const T* __restrict__ src, int64_t t0, int64_t n0,
                                        T* v) {
    const int t = threadIdx.x & 15, q = (threadIdx.x >> 4) & 3;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int64_t n = n0 + 4 * q + j;
        v[j] = t0 + t < p.len && n < p.state ? src[n * p.len + step_of(p, t0 + t)] : from_f32<T>(0.f);
    }
}
template <typename T>
__device__ __forceinline__ void store_bc(const T* raw, float* dst) {
    const int t = threadIdx.x & 15, q = (threadIdx.x >> 4) & 3;
    const float v[4] = {to_f32(raw[0]), to_f32(raw[1]), to_f32(raw[2]), to_f32(raw[3])};
    float* at = dst + t * kBcPitch + 4 * q;
    *reinterpret_cast<float4*>(at) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(at + kStates) = make_float4(v[1], v[0], v[3], v[2]);
    *reinterpret_cast<float4*>(at + 2 * kStates) = make_float4(v[2], v[3], v[0], v[1]);
    *reinterpret_cast<float4*>(at + 3 * kStates) = make_float4(v[3], v[2], v[1], v[0]);
}

// ---- activations: raw tiles copied ahead -----------------------------------
// A warp's raw tile of one tensor: 16 rows of 16 steps in memory order.
constexpr int kRawBytes = 4 * kWarpRows;
template <typename T>
__device__ __forceinline__ int raw_at(int row) {
    if constexpr (sizeof(T) == 4) return row_at(row);
    return row * 24 + (row >= 8 ? 16 : 0);
}

__device__ __forceinline__ uint32_t smem_addr(const void* v) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(v));
}

// Starts the copy of a warp's tile whose first step in memory is `ps` (it may
// reach outside the row: those elements are left alone).  src: the warp's
// first row.
template <typename T>
__device__ __forceinline__ void copy_rows(const T* __restrict__ src, int64_t len, int rows, int64_t ps, int width,
                                          T* dst) {
    const int lane = threadIdx.x & 31;
    if (width == 16) {
        constexpr int kV = 16 / sizeof(T), kC = kTile / kV;  // elements of a copy, copies of a row
#pragma unroll
        for (int i = 0; i < kRowsW * kC / 32; ++i) {
            const int row = (lane + 32 * i) / kC, c = (lane % kC) * kV;
            if (row < rows && ps + c >= 0 && ps + c < len)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(dst + raw_at<T>(row) + c)),
                             "l"(src + row * len + ps + c)
                             : "memory");
        }
    } else if (width == 4) {
        constexpr int kV = 4 / sizeof(T), kC = kTile / kV;
#pragma unroll
        for (int i = 0; i < kRowsW * kC / 32; ++i) {
            const int row = (lane + 32 * i) / kC, c = (lane % kC) * kV;
            if (row < rows && ps + c >= 0 && ps + c < len)
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_addr(dst + raw_at<T>(row) + c)),
                             "l"(src + row * len + ps + c)
                             : "memory");
        }
    } else {
#pragma unroll
        for (int i = 0; i < kRowsW * kTile / 32; ++i) {
            const int row = (lane + 32 * i) / kTile, c = lane % kTile;
            if (row < rows && ps + c >= 0 && ps + c < len) dst[raw_at<T>(row) + c] = src[row * len + ps + c];
        }
    }
}

// The four activations of a warp's tile.
template <typename T, typename TG, bool GRAD>
struct RawTile {
    T* u;
    T* delta;
    T* z;
    TG* dout;
    __device__ __forceinline__ RawTile(char (*buf)[kWarps][kRawBytes], int w)
        : u(reinterpret_cast<T*>(buf[0][w])), delta(reinterpret_cast<T*>(buf[1][w])),
          z(reinterpret_cast<T*>(buf[GRAD ? 2 : 0][w])), dout(reinterpret_cast<TG*>(buf[GRAD ? 3 : 0][w])) {}
    __device__ __forceinline__ void start(const M1BwdParams& p, const Plan& pl, const Lane& l, int64_t t0) const {
        const int64_t off = (l.b * p.dim + l.d0) * p.len;
        const int64_t ps = p.reverse ? p.len - kTile - t0 : t0;
        copy_rows(static_cast<const T*>(p.delta) + off, p.len, l.rows, ps, pl.width, delta);
        copy_rows(static_cast<const T*>(p.u) + off, p.len, l.rows, ps, pl.width, u);
        if (GRAD) {
            copy_rows(static_cast<const TG*>(p.dout) + off, p.len, l.rows, ps, pl.gwidth, dout);
            if (p.z) copy_rows(static_cast<const T*>(p.z) + off, p.len, l.rows, ps, pl.width, z);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    // Every lane's own copies, then everybody's; the `later` newest groups may
    // still be under way.
    template <int later>
    static __device__ __forceinline__ void wait() {
        asm volatile("cp.async.wait_group %0;" ::"n"(later) : "memory");
        __syncwarp();
    }
};

__device__ __forceinline__ float2 fadd2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 ra, rb, rd;\n\t"
        "mov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
        "add.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// A of a row slot's four states.  A decay is 2^(A (dt log2(e))): A itself stays
// exact, so that no rounding of the factor common to all of a row's steps adds up
// over them (at A = -1 .. -16 none is seen to: dA of 1 x 1536 rows of 32768 steps in 128
// segments is 1.2e-6 off with A log2(e) rounded, too).
__device__ __forceinline__ void load_a(const M1BwdParams& p, const Lane& l, int64_t n0, int k, float2* A) {
    float v[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const int64_t n = n0 + slot_state(l, s);
        v[s] = l.live(k) && n < p.state ? p.A[(l.d0 + l.row(k)) * p.state + n] : 0.f;
    }
    A[0] = make_float2(v[0], v[1]);
    A[1] = make_float2(v[2], v[3]);
}

// The same lane's values of a (batch, dim, state) tensor (null: zeros).
__device__ __forceinline__ void load_state(const M1BwdParams& p, const Lane& l, int64_t n0, int k, const float* src,
                                           float2* h) {
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (src && l.live(k)) {
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int64_t n = n0 + slot_state(l, s);
            if (n < p.state) v[s] = src[(l.b * p.dim + l.d0 + l.row(k)) * p.state + n];
        }
    }
    h[0] = make_float2(v[0], v[1]);
    h[1] = make_float2(v[2], v[3]);
}

__device__ __forceinline__ float4 join(const float2* v) { return make_float4(v[0].x, v[0].y, v[1].x, v[1].y); }
__device__ __forceinline__ void cut(const float4& v, float2* o) {
    o[0] = make_float2(v.x, v.y);
    o[1] = make_float2(v.z, v.w);
}
__device__ __forceinline__ void cut(const float4& v, float* o) {
    o[0] = v.x;
    o[1] = v.y;
    o[2] = v.z;
    o[3] = v.w;
}
__device__ __forceinline__ void store4(float* dst, const float4& v) { *reinterpret_cast<float4*>(dst) = v; }
__device__ __forceinline__ void store4(__nv_bfloat16* dst, const float4& v) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(dst) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

// 2^(x A) of four states.
__device__ __forceinline__ void decay(float x, const float2* A, float2* a) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        const float2 v = fmul2(both(x), A[s]);
        a[s] = make_float2(ex2_approx(v.x), ex2_approx(v.y));
    }
}

// ---- (1) forward sweep -----------------------------------------------------
// SPLIT: states start from zero in every segment, and the segment's aggregates
// (end state, gradient it would pass back, dt summed) are left for the carries.
template <typename T, typename TG, bool SPLIT>
__global__ void __launch_bounds__(kThreads, SPLIT ? 4 : 6) m1_bwd_sweep(M1BwdParams p, Plan pl, Ws ws, int64_t n0) {
    __shared__ __align__(16) float sB[kTile * kBcPitch];
    __shared__ __align__(16) float sC[SPLIT ? kTile * kBcPitch : 4];
    __shared__ __align__(16) float sDt[kWarps * kWarpRows];  // dt log2(e)
    __shared__ __align__(16) float sDu[kWarps * kWarpRows];
    __shared__ __align__(16) float sDy[SPLIT ? kWarps * kWarpRows : 4];
    __shared__ float sBias[kRowsC];
    __shared__ __align__(16) char sRaw[SPLIT ? 4 : 2][kWarps][kRawBytes];
    const Lane l = where(p, pl);
    const int w = threadIdx.x / 32;
    float2 A[2][2], h[2][2], prod[2][2], gl[2][2];
    int at[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        load_a(p, l, n0, k, A[k]);
        load_state(p, l, n0, k, SPLIT ? nullptr : p.h0, h[k]);
        prod[k][0] = prod[k][1] = both(1.f);
        gl[k][0] = gl[k][1] = both(0.f);
        at[k] = w * kWarpRows + row_at(l.row(k));
    }
    float sdt = 0.f;  // of row slot 0
    const bool has_bc = threadIdx.x < 64 || SPLIT;
    const T* src = static_cast<const T*>(threadIdx.x < 64 ? p.B : p.C) + (l.b * p.groups + l.g) * p.state * p.len;
    float* bc = SPLIT && threadIdx.x >= 64 ? sC : sB;
    if (l.lane < kRowsW)
        sBias[w * kRowsW + l.lane] = p.delta_bias && l.lane < l.rows ? p.delta_bias[l.d0 + l.lane] : 0.f;
    const float* bs = sB + (l.r & 3) * kStates + 4 * l.q;
    const float* cs = sC + (SPLIT ? (l.r & 3) * kStates + 4 * l.q : 0);
    // elementwise part: half a warp takes a row's 16 steps, eight rows in turn
    const int step = l.lane & 15, half = l.lane >> 4, ph = p.reverse ? kTile - 1 - step : step;
    const int rows = l.rows - 8 * half;
    const RawTile<T, TG, SPLIT> raw(sRaw, w);
    const int64_t tile0 = l.seg * pl.seg_tiles, tile1 = min(tile0 + pl.seg_tiles, pl.tiles);
    T bcv[4];
    raw.start(p, pl, l, tile0 * kTile);
    if (has_bc) load_bc<T>(p, src, tile0 * kTile, n0, bcv);
    int64_t gb = l.warp_id * pl.blocks + tile0 * kTileBlocks;
    for (int64_t tile = tile0; tile < tile1; ++tile) {
        const int64_t t0 = tile * kTile;
        const bool on = t0 + step < p.len;
        raw.template wait<0>();
        auto elementwise = [&](auto softplus, auto gated) {
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                const int row = 8 * half + r, o = w * kWarpRows + row_at(row) + step;
                // a step or row that is not there: decay 1, nothing added
                const bool there = on && r < rows;
                float dt, slope;
                dt_of<softplus.value>(to_f32(raw.delta[raw_at<T>(row) + ph]) + sBias[w * kRowsW + row], &dt, &slope);
                sDt[o] = there ? dt * kLog2e : 0.f;
                sDu[o] = there ? dt * to_f32(raw.u[raw_at<T>(row) + ph]) : 0.f;
                if (SPLIT) {
                    float dy = to_f32(raw.dout[raw_at<TG>(row) + ph]);
                    if (gated.value) dy *= silu_fast(to_f32(raw.z[raw_at<T>(row) + ph]));
                    sDy[o] = there ? dy : 0.f;
                }
            }
        };
        with_flags(p, elementwise);
        __syncthreads();  // every warp is done with the last tile's B and C
        if (has_bc) store_bc<T>(bcv, bc);
        if (tile + 1 < tile1) {
            raw.start(p, pl, l, t0 + kTile);
            if (has_bc) load_bc<T>(p, src, t0 + kTile, n0, bcv);
        }
        __syncthreads();
#pragma unroll 1
        for (int blk = 0; blk < kTileBlocks; ++blk, ++gb) {
            const int t4 = blk * kT;
            float dt[2][4], du[2][4], dy[2][4];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                ws.ckpt[gb * 64 + k * 32 + l.lane] = join(h[k]);
                cut(*reinterpret_cast<const float4*>(sDt + at[k] + t4), dt[k]);
                cut(*reinterpret_cast<const float4*>(sDu + at[k] + t4), du[k]);
                if (SPLIT) cut(*reinterpret_cast<const float4*>(sDy + at[k] + t4), dy[k]);
            }
            if (SPLIT && !(l.q & 1)) ws.sdt[gb * kRowsW + l.row(0)] = sdt;
#pragma unroll
            for (int i = 0; i < kT; ++i) {
                float2 B[2], C[2];
                cut(*reinterpret_cast<const float4*>(bs + (t4 + i) * kBcPitch), B);
                if (SPLIT) {
                    cut(*reinterpret_cast<const float4*>(cs + (t4 + i) * kBcPitch), C);
                    sdt += dt[0][i];
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    float2 a[2];
                    decay(dt[k][i], A[k], a);
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        h[k][s] = ffma2(a[s], h[k][s], fmul2(both(du[k][i]), B[s]));
                        if (SPLIT) {
                            prod[k][s] = fmul2(prod[k][s], a[s]);
                            gl[k][s] = ffma2(prod[k][s], fmul2(both(dy[k][i]), C[s]), gl[k][s]);
                        }
                    }
                }
            }
        }
    }
    griddep_launch_dependents();
    if (SPLIT) {
        const int64_t agg = l.seg * pl.units * kWarps + l.warp_id;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            ws.hend[agg * 64 + k * 32 + l.lane] = join(h[k]);
            ws.gend[agg * 64 + k * 32 + l.lane] = join(gl[k]);
        }
        if (!(l.q & 1)) ws.stot[agg * kRowsW + l.row(0)] = sdt;
    }
}

// ---- (2) carries over a row's segments -------------------------------------
// hend[s] becomes the state entering segment s, gend[s] the gradient entering
// it from segment s + 1 (dL/dh at its last step, without that step's own dy C).
__global__ void __launch_bounds__(kThreads) m1_bwd_carry(M1BwdParams p, Plan pl, Ws ws, int64_t n0) {
    const Lane l = where(p, pl);  // grid: units x 4 CTAs, per row slot and direction
    const int k = static_cast<int>(l.seg) & 1;
    const bool back = l.seg >= 2;
    float2 A[2], h[2], a[2], e[2];
    load_a(p, l, n0, k, A);
    load_state(p, l, n0, k, back ? p.dlast : p.h0, h);
    griddep_wait();  // the sweep's aggregates
    griddep_launch_dependents();
    const int64_t stride = pl.units * kWarps;
    float4* const ends = (back ? ws.gend : ws.hend) + l.warp_id * 64 + k * 32 + l.lane;
    const float* const sums = ws.stot + l.warp_id * kRowsW + l.row(k);
    constexpr int kAhead = 16;  // segments whose aggregates are loaded together
    for (int64_t s0 = 0; s0 < pl.segs; s0 += kAhead) {
        float4 v[kAhead];
        float sd[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int64_t i = min(s0 + j, pl.segs - 1), at = (back ? pl.segs - 1 - i : i) * stride;
            v[j] = ends[at * 64];
            sd[j] = sums[at * kRowsW];
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int64_t i = s0 + j;
            if (i >= pl.segs) break;
            ends[(back ? pl.segs - 1 - i : i) * stride * 64] = join(h);
            decay(sd[j], A, a);
            cut(v[j], e);
            h[0] = ffma2(a[0], h[0], e[0]);
            h[1] = ffma2(a[1], h[1], e[1]);
        }
    }
}

// ---- (3) main kernel -------------------------------------------------------
constexpr int kRedPitch = kTile + 4;  // floats between states of a warp's dB / dC tile
struct MainSmem {
    float B[kTile * kBcPitch], C[kTile * kBcPitch];
    float dt[kWarps * kWarpRows];     // dt, then du
    float u[kWarps * kWarpRows];
    float dy[kWarps * kWarpRows];
    float fz[kWarps * kWarpRows];     // dout s (1 + z (1 - s)), then dz
    float slope[kWarps * kWarpRows];  // ddt/dx, then ddelta
    float4 hin[2][kThreads];          // state entering the segment
    float4 ck[2][kThreads];           // the next block's saved state
    float dB[kWarps][kStates * kRedPitch];
    float dC[kWarps][kStates * kRedPitch];
    float bias[kRowsC];
    char raw[4][kWarps][kRawBytes];
};

// First two stages of the sum over a warp's rows of one step's four state
// slots (already summed over the lane's two rows): the lane ends with state
// 4q + (r & 3) summed over rows differing in bits 0 and 1.
__device__ __forceinline__ float rows_stage(const float2* v) {
    const float2 a = fadd2(v[0], make_float2(__shfl_xor_sync(0xffffffffu, v[1].x, 8),
                                             __shfl_xor_sync(0xffffffffu, v[1].y, 8)));
    return a.x + __shfl_xor_sync(0xffffffffu, a.y, 4);
}

// Last stage, over row bit 2, for the four steps of a block: rows 0-3 keep
// steps 0 and 1, rows 4-7 steps 2 and 3, and store them.
__device__ __forceinline__ void rows_store(const Lane& l, const float* v, float* dst) {
    const bool hi = l.r & 4;
    float2 k;
    k.x = (hi ? v[2] : v[0]) + __shfl_xor_sync(0xffffffffu, hi ? v[0] : v[2], 16);
    k.y = (hi ? v[3] : v[1]) + __shfl_xor_sync(0xffffffffu, hi ? v[1] : v[3], 16);
    *reinterpret_cast<float2*>(dst + (4 * l.q + (l.r & 3)) * kRedPitch + (hi ? 2 : 0)) = k;
}

// Sum over a row's four lanes of the block's per-step values of both row
// slots: lane q ends with row slot 0 (row r + 8 (q >> 1)), steps 2 (q & 1) and
// the one after.
__device__ __forceinline__ float2 lanes_sum(const Lane& l, const float (*v)[kT]) {
    float k[kT];
#pragma unroll
    for (int i = 0; i < kT; ++i) k[i] = v[0][i] + __shfl_xor_sync(0xffffffffu, v[1][i], 2);
    const bool b = l.q & 1;
    float2 o;
    o.x = (b ? k[2] : k[0]) + __shfl_xor_sync(0xffffffffu, b ? k[0] : k[2], 1);
    o.y = (b ? k[3] : k[1]) + __shfl_xor_sync(0xffffffffu, b ? k[1] : k[3], 1);
    return o;
}

template <typename T, typename TG>
__global__ void __launch_bounds__(kThreads, kCtasSm) m1_bwd_main(M1BwdParams p, Plan pl, Ws ws, int64_t n0, int first,
                                                                 int last) {
    extern __shared__ __align__(16) char raw_smem[];
    MainSmem& sm = *reinterpret_cast<MainSmem*>(raw_smem);
    const Lane l = where(p, pl);
    const int w = threadIdx.x / 32;
    const int64_t agg = l.seg * pl.units * kWarps + l.warp_id;
    const bool split = pl.segs > 1;
    float2 A[2][2], ag[2][2], dA[2][2];
    int at[2];
    griddep_wait();  // the sweep's states, the carries
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        load_a(p, l, n0, k, A[k]);
        if (split) {
            cut(ws.gend[agg * 64 + k * 32 + l.lane], ag[k]);
            sm.hin[k][threadIdx.x] = ws.hend[agg * 64 + k * 32 + l.lane];
        } else {
            load_state(p, l, n0, k, p.dlast, ag[k]);
        }
        dA[k][0] = dA[k][1] = both(0.f);
        at[k] = w * kWarpRows + row_at(l.row(k));
    }
    const float Dskip = p.d_skip && l.live(0) ? p.d_skip[l.d0 + l.row(0)] : 0.f;
    float dD = 0.f, dbias = 0.f;  // of row slot 0, the lane's two steps of each block
    const int64_t bg = l.b * p.groups + l.g;
    const T* src = static_cast<const T*>(threadIdx.x < 64 ? p.B : p.C) + bg * p.state * p.len;
    if (l.lane < kRowsW)
        sm.bias[w * kRowsW + l.lane] = p.delta_bias && l.lane < l.rows ? p.delta_bias[l.d0 + l.lane] : 0.f;
    __syncwarp();
    const float* bs = sm.B + (l.r & 3) * kStates + 4 * l.q;
    const float* cs = sm.C + (l.r & 3) * kStates + 4 * l.q;
    // elementwise parts: half a warp takes a row's 16 steps, eight rows in turn
    const int step = l.lane & 15, half = l.lane >> 4, ph = p.reverse ? kTile - 1 - step : step;
    const int64_t row0 = (l.b * p.dim + l.d0 + 8 * half) * p.len;
    const int rows = l.rows - 8 * half;
    const RawTile<T, TG, true> raw(sm.raw, w);
    const int64_t tile0 = l.seg * pl.seg_tiles, tile1 = min(tile0 + pl.seg_tiles, pl.tiles);
    const int64_t plane = p.batch * p.dim * p.len;
    T bcv[4];
    raw.start(p, pl, l, (tile1 - 1) * kTile);
    load_bc<T>(p, src, (tile1 - 1) * kTile, n0, bcv);
    // the blocks' saved states, copied a block ahead, and dt sums (lane i holds
    // values i and 32 + i of the tile's [4 blocks][16 rows]), a tile ahead
    const int64_t gb_end = l.warp_id * pl.blocks + tile0 * kTileBlocks;
    int64_t gb = l.warp_id * pl.blocks + tile1 * kTileBlocks - 1;
    auto start_ck = [&] {
#pragma unroll
        for (int k = 0; k < 2; ++k)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(&sm.ck[k][threadIdx.x])),
                         "l"(ws.ckpt + gb * 64 + k * 32 + l.lane)
                         : "memory");
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    float sd_next[2] = {0.f, 0.f};
    auto load_sd = [&](int64_t tile) {
        const float* at = ws.sdt + (l.warp_id * pl.blocks + tile * kTileBlocks) * kRowsW + l.lane;
        sd_next[0] = at[0];
        sd_next[1] = at[32];
    };
    start_ck();
    if (split) load_sd(tile1 - 1);
    for (int64_t tile = tile1 - 1; tile >= tile0; --tile) {
        const int64_t t0 = tile * kTile;
        const bool on = t0 + step < p.len;
        raw.template wait<1>();  // the newest group is a saved state's
        auto elementwise = [&](auto softplus, auto gated) {
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                const int row = 8 * half + r, o = w * kWarpRows + row_at(row) + step;
                // a step or row that is not there: decay 1, no gradient
                const bool there = on && r < rows;
                float dt, slope, dy = to_f32(raw.dout[raw_at<TG>(row) + ph]), fz = 0.f;
                dt_of<softplus.value>(to_f32(raw.delta[raw_at<T>(row) + ph]) + sm.bias[w * kRowsW + row], &dt, &slope);
                if (gated.value) {
                    const float z = to_f32(raw.z[raw_at<T>(row) + ph]);
                    const float s = rcp_approx(1.f + ex2_approx(-z * kLog2e));
                    fz = dy * s * fmaf(z, 1.f - s, 1.f);
                    dy *= z * s;
                }
                sm.dt[o] = there ? dt : 0.f;
                sm.slope[o] = there ? slope : 0.f;
                sm.u[o] = there ? to_f32(raw.u[raw_at<T>(row) + ph]) : 0.f;
                sm.dy[o] = there ? dy : 0.f;
                sm.fz[o] = fz;
            }
        };
        with_flags(p, elementwise);
        store_bc<T>(bcv, threadIdx.x < 64 ? sm.B : sm.C);
        __syncthreads();
        const float sd_tile[2] = {sd_next[0], sd_next[1]};
        if (tile > tile0) {
            raw.start(p, pl, l, t0 - kTile);
            load_bc<T>(p, src, t0 - kTile, n0, bcv);
            if (split) load_sd(tile - 1);
        }
#pragma unroll 1
        for (int blk = kTileBlocks - 1; blk >= 0; --blk) {
            float2 h[2][2];
            // each lane reads back what it copied itself.  At a tile's first block
            // the activations' copies, started since, may still be under way.
            if (blk == kTileBlocks - 1 && tile > tile0) asm volatile("cp.async.wait_group 1;" ::: "memory");
            else asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                cut(sm.ck[k][threadIdx.x], h[k]);
                if (split) {
                    const float sd = __shfl_sync(0xffffffffu, blk & 2 ? sd_tile[1] : sd_tile[0], (blk & 1) * kRowsW + l.row(k));
                    float2 a[2], in[2];
                    decay(sd, A[k], a);
                    cut(sm.hin[k][threadIdx.x], in);
                    h[k][0] = ffma2(a[0], in[0], h[k][0]);
                    h[k][1] = ffma2(a[1], in[1], h[k][1]);
                }
            }
            if (gb > gb_end) {
                --gb;
                start_ck();
            }
            const float* bb = bs + blk * kT * kBcPitch;
            const float* cb = cs + blk * kT * kBcPitch;
            float dt[2][kT], dy[2][kT], du[2][kT];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int o = at[k] + blk * kT;
                float u[kT];
                cut(*reinterpret_cast<const float4*>(sm.dt + o), dt[k]);
                cut(*reinterpret_cast<const float4*>(sm.dy + o), dy[k]);
                cut(*reinterpret_cast<const float4*>(sm.u + o), u);
#pragma unroll
                for (int i = 0; i < kT; ++i) du[k][i] = dt[k][i] * u[i];
            }
            float2 a[kT][2][2], ah[kT][2][2];
            float part[2][kT], vr[kT];
            // forward through the block
#pragma unroll
            for (int i = 0; i < kT; ++i) {
                float2 B[2], C[2], dc[2];
                cut(*reinterpret_cast<const float4*>(bb + i * kBcPitch), B);
                cut(*reinterpret_cast<const float4*>(cb + i * kBcPitch), C);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    float2 y;
                    decay(dt[k][i] * kLog2e, A[k], a[i][k]);
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        ah[i][k][s] = fmul2(a[i][k][s], h[k][s]);
                        h[k][s] = ffma2(both(du[k][i]), B[s], ah[i][k][s]);
                        y = s ? ffma2(C[s], h[k][s], y) : fmul2(C[s], h[k][s]);
                        dc[s] = k ? ffma2(both(dy[k][i]), h[k][s], dc[s]) : fmul2(both(dy[k][i]), h[k][s]);
                    }
                    part[k][i] = y.x + y.y;
                }
                vr[i] = rows_stage(dc);
            }
            rows_store(l, vr, sm.dC[w] + blk * kT);
            float2 y2 = lanes_sum(l, part);
            // gradient back through the block
            float part2[2][kT];
            float2 dAb[2][2];  // the block's share of dA: short sums first
#pragma unroll
            for (int i = kT - 1; i >= 0; --i) {
                float2 B[2], C[2], db[2];
                cut(*reinterpret_cast<const float4*>(bb + i * kBcPitch), B);
                cut(*reinterpret_cast<const float4*>(cb + i * kBcPitch), C);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    float2 sb, sa;
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        const float2 g = ffma2(both(dy[k][i]), C[s], ag[k][s]);
                        const float2 gah = fmul2(g, ah[i][k][s]);
                        sb = s ? ffma2(g, B[s], sb) : fmul2(g, B[s]);
                        sa = s ? ffma2(gah, A[k][s], sa) : fmul2(gah, A[k][s]);
                        dAb[k][s] = i == kT - 1 ? fmul2(gah, both(dt[k][i])) : ffma2(gah, both(dt[k][i]), dAb[k][s]);
                        db[s] = k ? ffma2(g, both(du[k][i]), db[s]) : fmul2(g, both(du[k][i]));
                        ag[k][s] = fmul2(a[i][k][s], g);
                    }
                    part[k][i] = sb.x + sb.y;
                    part2[k][i] = sa.x + sa.y;
                }
                vr[i] = rows_stage(db);
            }
            rows_store(l, vr, sm.dB[w] + blk * kT);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                dA[k][0] = fadd2(dA[k][0], dAb[k][0]);
                dA[k][1] = fadd2(dA[k][1], dAb[k][1]);
            }
            float2 sb2 = lanes_sum(l, part), sa2 = lanes_sum(l, part2);
            // the lane's two steps of row slot 0; du takes the place of dt, which
            // the row's other lanes have read by now
            __syncwarp();
            const int o = at[0] + blk * kT + 2 * (l.q & 1);
            if (!first || !last) {
                // states beyond 16: sums over the state blocks so far
                float* sums[3] = {&y2.x, &sb2.x, &sa2.x};
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int64_t t = t0 + blk * kT + 2 * (l.q & 1) + e;
                    if (!l.live(0) || t >= p.len) continue;
                    float* acc = ws.acc + (l.b * p.dim + l.d0 + l.row(0)) * p.len + t;
#pragma unroll
                    for (int m = 0; m < 3; ++m) {
                        if (!first) sums[m][e] += acc[m * plane];
                        if (!last) acc[m * plane] = sums[m][e];
                    }
                }
            }
            const float2 u = *reinterpret_cast<const float2*>(sm.u + o), g = *reinterpret_cast<const float2*>(sm.dy + o);
            const float2 t2 = *reinterpret_cast<const float2*>(sm.dt + o);
            float2* fz = reinterpret_cast<float2*>(sm.fz + o);
            float2* sl = reinterpret_cast<float2*>(sm.slope + o);
            const float2 dx = fmul2(ffma2(u, sb2, sa2), *sl);
            *fz = fmul2(*fz, ffma2(both(Dskip), u, y2));
            *sl = dx;
            *reinterpret_cast<float2*>(sm.dt + o) = ffma2(both(Dskip), g, fmul2(t2, sb2));
            dD = fmaf(g.x, u.x, fmaf(g.y, u.y, dD));
            dbias += dx.x + dx.y;
        }
        __syncthreads();
        if (last) {
            const int64_t wrow0 = (l.b * p.dim + l.d0) * p.len;
            auto copy_out = [&](const float* from, void* to) {
                if (pl.width_out == 16) {
                    // four steps a lane, eight rows at once
                    const int c = (l.lane & 3) * 4;
                    const int64_t t = p.reverse ? p.len - 4 - (t0 + c) : t0 + c;
                    T* dst = static_cast<T*>(to) + wrow0 + (l.lane >> 2) * p.len + t;
                    const float* at = from + w * kWarpRows + (l.lane >> 2) * kRowPitch + c;
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        float4 v = *reinterpret_cast<const float4*>(at + k * (8 * kRowPitch + kUpper));
                        if (p.reverse) v = make_float4(v.w, v.z, v.y, v.x);
                        if ((l.lane >> 2) + 8 * k < l.rows && t0 + c < p.len) store4(dst + 8 * k * p.len, v);
                    }
                } else {
                    T* dst = static_cast<T*>(to) + row0 + step_of(p, t0 + step);
                    const float* at = from + w * kWarpRows + row_at(8 * half) + step;
#pragma unroll
                    for (int r = 0; r < 8; ++r, dst += p.len)
                        if (on && r < rows) *dst = from_f32<T>(at[r * kRowPitch]);
                }
            };
            copy_out(sm.dt, p.du);
            copy_out(sm.slope, p.ddelta);
            if (p.z) copy_out(sm.fz, p.dz);
        }
        // dB and dC of the tile, four steps a thread: the warps' sums in order
        static_assert(2 * kStates * kTile == 4 * kThreads);
        const int t = (threadIdx.x & 3) * 4, n = (threadIdx.x >> 2) & 15;
        float2 v[2] = {both(0.f), both(0.f)};
#pragma unroll
        for (int k = 0; k < kWarps; ++k) {
            float2 x[2];
            cut(*reinterpret_cast<const float4*>((threadIdx.x < 64 ? sm.dB[k] : sm.dC[k]) + n * kRedPitch + t), x);
            v[0] = fadd2(v[0], x[0]);
            v[1] = fadd2(v[1], x[1]);
        }
        *reinterpret_cast<float4*>((threadIdx.x < 64 ? ws.dbp : ws.dcp) + (l.unit * kStates + n) * pl.tiles * kTile +
                                   t0 + t) = join(v);
    }
    griddep_launch_dependents();
#pragma unroll
    for (int k = 0; k < 2; ++k) ws.dap[agg * 64 + k * 32 + l.lane] = join(dA[k]);
    if (last) {
        dD += __shfl_xor_sync(0xffffffffu, dD, 1);
        dbias += __shfl_xor_sync(0xffffffffu, dbias, 1);
        if (!(l.q & 1)) {
            ws.ddp[agg * kRowsW + l.row(0)] = dD;
            ws.dbiasp[agg * kRowsW + l.row(0)] = dbias;
        }
    }
    if (p.dh0 && l.seg == 0) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const float4 v4 = join(ag[k]);
            const float v[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int64_t n = n0 + slot_state(l, s);
                if (l.live(k) && n < p.state) p.dh0[(l.b * p.dim + l.d0 + l.row(k)) * p.state + n] = v[s];
            }
        }
    }
}

// ---- (4) partial sums ------------------------------------------------------
// CTAs 0 .. row_ctas - 1 (first: they take longest): 16 rows' dA, dD and dbias over
// batch and segments, a thread per (row slot, lane) of the main kernel's warp; the
// partials of a channel are added kSlices apart, then the kSlices sums.  The rest:
// dB and dC, a thread adds four steps' partials over the group's row blocks.
constexpr int kRedThreads = 512, kSlices = kRedThreads / 64;
template <typename T>
__global__ void __launch_bounds__(kRedThreads) m1_bwd_reduce(M1BwdParams p, Plan pl, Ws ws, int64_t n0, int last,
                                                             int64_t row_ctas) {
    const int64_t states = min(static_cast<int64_t>(kStates), p.state - n0);
    griddep_wait();  // the main kernel's partial sums
    if (blockIdx.x >= row_ctas) {
        // four steps a thread; the partials are padded to whole tiles
        const int64_t padded = pl.tiles * kTile, quads = padded / 4, nq = p.batch * p.groups * states * quads;
        int64_t i = (static_cast<int64_t>(blockIdx.x) - row_ctas) * kRedThreads + threadIdx.x;
        if (i >= 2 * nq) return;
        const bool is_c = i >= nq;
        i -= is_c ? nq : 0;
        int64_t bgn, bg, n, t4;
        divide(i, quads, &bgn, &t4);
        divide(bgn, states, &bg, &n);
        const float* src = (is_c ? ws.dcp : ws.dbp) + (bg * pl.rblocks * kStates + n) * padded + 4 * t4;
        float2 v[2] = {both(0.f), both(0.f)};
#pragma unroll 8
        for (int64_t k = 0; k < pl.rblocks; ++k) {
            float2 x[2];
            cut(*reinterpret_cast<const float4*>(src + k * kStates * padded), x);
            v[0] = fadd2(v[0], x[0]);
            v[1] = fadd2(v[1], x[1]);
        }
        T* dst = static_cast<T*>(is_c ? p.dC : p.dB) + (bg * p.state + n0 + n) * p.len;
        const float o[4] = {v[0].x, v[0].y, v[1].x, v[1].y};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (4 * t4 + e < p.len) dst[step_of(p, 4 * t4 + e)] = from_f32<T>(o[e]);
        return;
    }
    __shared__ float4 sum[kSlices][64];
    __shared__ float sumd[kSlices][2 * kRowsW];
    const int64_t wg = blockIdx.x % (pl.rblocks * kWarps), g = blockIdx.x / (pl.rblocks * kWarps);
    const int64_t parts = pl.segs * p.batch, row0 = g * pl.rblocks * kWarps + wg, rows = p.groups * pl.rblocks * kWarps;
    const int slice = threadIdx.x / 64, i = threadIdx.x % 64;
    // partial k: segment k / batch of batch k % batch
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    float d = 0.f;
#pragma unroll 8
    for (int64_t k = slice; k < parts; k += kSlices) {
        const int64_t at = k * rows + row0;
        const float4 x = ws.dap[at * 64 + i];
        v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
        if (last && i < 2 * kRowsW) d += (i < kRowsW ? ws.ddp : ws.dbiasp)[at * kRowsW + i % kRowsW];
    }
    sum[slice][i] = v;
    if (i < 2 * kRowsW) sumd[slice][i] = d;
    __syncthreads();
    if (slice) return;
#pragma unroll
    for (int k = 1; k < kSlices; ++k) {
        const float4 x = sum[k][i];
        v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
        if (i < 2 * kRowsW) d += sumd[k][i];
    }
    // the slots of the lane that wrote it: see Lane::row and slot_state
    const int slot = i / 32, lane = i % 32, q = lane & 3, r = lane >> 2, row = r + 8 * (slot ^ (q >> 1));
    const float o[4] = {v.x, v.y, v.z, v.w};
    if (wg * kRowsW + row < pl.per)
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int64_t n = n0 + 4 * q + (s ^ (r & 3));
            if (n < p.state) p.dA[(g * pl.per + wg * kRowsW + row) * p.state + n] = o[s];
        }
    if (last && i < 2 * kRowsW && wg * kRowsW + i % kRowsW < pl.per) {
        float* out = i < kRowsW ? p.dD : p.ddelta_bias;
        if (out) out[g * pl.per + wg * kRowsW + i % kRowsW] = d;
    }
}

template <typename T, typename TG>
cudaError_t run(const M1BwdParams& p, const Plan& pl, const Ws& ws, cudaStream_t stream) {
    cudaError_t e = cudaFuncSetAttribute(m1_bwd_main<T, TG>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(sizeof(MainSmem)));
    if (e != cudaSuccess) return e;
    const unsigned grid = static_cast<unsigned>(pl.units * pl.segs);
    for (int64_t n0 = 0; n0 < p.state; n0 += kStates) {
        const int first = n0 == 0, last = n0 + kStates >= p.state;
        // The kernels after the sweep are launched when their predecessors' CTAs come
        // to their end (and wait for it before they read what they wrote).  Launched
        // earlier, few CTAs of the main kernel are packed on the SMs that have room:
        // 1464 us instead of 1187 with one segment of 8 x 1536 rows.
        if (pl.segs > 1) {
            m1_bwd_sweep<T, TG, true><<<grid, kThreads, 0, stream>>>(p, pl, ws, n0);
            note_launch();
            e = cudaGetLastError();
            if (e != cudaSuccess) return e;
            e = launch_pdl(m1_bwd_carry, static_cast<unsigned>(4 * pl.units), kThreads, stream, p, pl, ws, n0);
        } else {
            m1_bwd_sweep<T, TG, false><<<grid, kThreads, 0, stream>>>(p, pl, ws, n0);
            e = cudaGetLastError();
        }
        note_launch();
        if (e != cudaSuccess) return e;
        e = launch_pdl_smem(m1_bwd_main<T, TG>, grid, kThreads, sizeof(MainSmem), stream, p, pl, ws, n0, first, last);
        note_launch();
        if (e != cudaSuccess) return e;
        const int64_t states = std::min<int64_t>(kStates, p.state - n0);
        const int64_t bc_ctas =
            (2 * p.batch * p.groups * states * pl.tiles * (kTile / 4) + kRedThreads - 1) / kRedThreads;
        const int64_t row_ctas = p.groups * pl.rblocks * kWarps;
        e = launch_pdl(m1_bwd_reduce<T>, static_cast<unsigned>(row_ctas + bc_ctas), kRedThreads, stream, p, pl, ws, n0,
                       last, row_ctas);
        note_launch();
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

}  // namespace

size_t m1_bwd_workspace_bytes(const M1BwdParams& p) { return make_ws(p, make_plan(p), nullptr).floats * sizeof(float); }

cudaError_t m1_bwd_launch(const M1BwdParams& p, void* workspace, cudaStream_t stream) {
    const Plan pl = make_plan(p);
    const int64_t most = (int64_t(1) << 31) - 1;
    if (pl.units * std::max<int64_t>(pl.segs, 4) > most || p.batch * p.groups * kStates * p.len / 64 + pl.units * kWarps > most) return cudaErrorInvalidValue;
    const Ws ws = make_ws(p, pl, workspace);
    if (p.dtype == kF32) {
        if (p.dout_dtype != kF32) return cudaErrorInvalidValue;
        return run<float, float>(p, pl, ws, stream);
    }
    return p.dout_dtype == kF32 ? run<__nv_bfloat16, float>(p, pl, ws, stream)
                                : run<__nv_bfloat16, __nv_bfloat16>(p, pl, ws, stream);
}

}  // namespace b200scan
