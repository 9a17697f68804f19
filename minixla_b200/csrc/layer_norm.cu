// Layer norm and its backward pass (mxb_layer_norm, mxb_layer_norm_backward).
//
// Forward, row by row: mean = sum(x) / C, var = sum((x - mean)^2) / C,
// rstd = 1 / sqrt(var + eps), y = (x - mean) * rstd * gamma + beta.
// Backward, with v = dy * gamma and xhat = (x - mean) * rstd:
//   dx = rstd * (v - sum(v) / C - xhat * sum(v * xhat) / C),
//   dgamma = sum over rows of dy * xhat, dbeta = sum over rows of dy.
// Everything is fp32; the variance is taken around the mean (a second pass
// over the registers), never as a difference of two large sums.
//
// Bound by HBM: x in, y out (backward: x and dy in, dx out), each once.  A
// row is held in registers between its sums and its output, by one warp up
// to 1024 columns and by a block beyond; only rows longer than a block can
// hold are read again (from L2).  A block's rows arrive through a ring in shared
// memory that bulk copies keep full: with loads by the threads themselves,
// which can only be issued between a row's two barriers, the same kernels
// reached 5.3 (forward) and 5.4 TB/s (backward); with the ring forward takes
// 86 us at 16384 x 4096 (6.2 TB/s) and backward 131 us at 8192 x 8192 (6.1
// TB/s), against 6.5 TB/s for a copy.  Short or odd rows are latency and
// instructions: 25 us for the backward pass of 5003 x 1027, of which its bytes need 9.  The
// gradients of gamma and beta are summed per thread over the rows its block
// walks through, then stored as one partial row per block and summed by a
// second small kernel in block order, so the result does not depend on timing.
#include "gemm_common.cuh"

#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <exception>

#include "runtime_internal.h"

namespace mxb {

namespace {

struct NormParams {
    const float* x;
    long long ldx;
    const float* gamma;
    const float* beta;
    float eps;
    float* y;
    long long ldy;
    float* mean;
    float* rstd;
    long long rows;
    int cols;
    unsigned long long timeout_ns;
    int* err;
};

struct NormGradParams {
    const float* dy;
    long long lddy;
    const float* x;
    long long ldx;
    const float* gamma;
    const float* mean;
    const float* rstd;
    float* dx;
    long long lddx;
    float* partial;   // [block][2][cols]: dgamma, dbeta (nullptr: neither is wanted)
    long long rows;
    int cols;
    unsigned long long timeout_ns;
    int* err;
};

// Accesses under a predicate, for rows of single floats (W = 1): the compiler puts a branch around a conditional asm
// statement, one for every access there (backward 20003 x 1027 74 -> 64 us without them, 2000 x 5001 42 -> 35).  Rows of
// four have few such accesses, and keep the branch.
__device__ __forceinline__ float load_if(bool wanted, const float* p, float otherwise) {
    float v = otherwise;
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\t@p ld.global.cs.f32 %0, [%1];\n\t}"
                 : "+f"(v)
                 : "l"(p), "r"(static_cast<int>(wanted))
                 : "memory");
    return v;
}
__device__ __forceinline__ void store_if(bool wanted, float* p, float v) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\t@p st.global.cs.f32 [%0], %1;\n\t}" ::"l"(p), "f"(v),
                 "r"(static_cast<int>(wanted))
                 : "memory");
}
__device__ __forceinline__ float load_shared_if(bool wanted, uint32_t addr, float otherwise) {
    float v = otherwise;
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\t@p ld.shared.f32 %0, [%1];\n\t}"
                 : "+f"(v)
                 : "r"(addr), "r"(static_cast<int>(wanted))
                 : "memory");
    return v;
}

// W consecutive floats at p + c, `past` from column `cols` on.
template <int W>
__device__ __forceinline__ void load_unit(float (&v)[W], const float* p, int c, int cols, float past = 0.0f) {
    if (W == 4 && c + W <= cols) {
        const float4 t = __ldcs(reinterpret_cast<const float4*>(p + c));
        v[0] = t.x;
        v[W > 1 ? 1 : 0] = t.y;
        v[W > 2 ? 2 : 0] = t.z;
        v[W > 3 ? 3 : 0] = t.w;
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = W == 1 ? load_if(c < cols, p + c, past) : c + i < cols ? __ldcs(p + c + i) : past;
    }
}

// The same for a vector that every row reads (gamma, beta): cached; `absent` where there is none.  EARLY: in a kernel
// that launch_early starts; elsewhere a read-only load, which the compiler may repeat for every row instead of keeping
// its result in a register that the kernel needs more (the backward pass of 5003 x 1027 is 7 us slower with the result pinned).
template <int W, bool EARLY>
__device__ __forceinline__ void load_param(float (&v)[W], const float* p, int c, int cols, float absent) {
    if (!p) {
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = absent;
    } else if (W == 4 && c + W <= cols) {
        const float4* at = reinterpret_cast<const float4*>(p + c);
        const float4 t = EARLY ? ld_global(at) : __ldg(at);
        v[0] = t.x;
        v[W > 1 ? 1 : 0] = t.y;
        v[W > 2 ? 2 : 0] = t.z;
        v[W > 3 ? 3 : 0] = t.w;
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = c + i < cols ? (EARLY ? ld_global(p + c + i) : __ldg(p + c + i)) : 0.0f;
    }
}

template <int W>
__device__ __forceinline__ void store_unit(const float (&v)[W], float* p, int c, int cols) {
    if (W == 4 && c + W <= cols) {
        __stcs(reinterpret_cast<float4*>(p + c), make_float4(v[0], v[W > 1 ? 1 : 0], v[W > 2 ? 2 : 0], v[W > 3 ? 3 : 0]));
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i)
            if (W == 1) {
                store_if(c < cols, p + c, v[0]);
            } else if (c + i < cols) {
                __stcs(p + c + i, v[i]);
            }
    }
}

__device__ __forceinline__ float2 warp_sum(float2 s) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        s.x += __shfl_xor_sync(0xffffffffu, s.x, o);
        s.y += __shfl_xor_sync(0xffffffffu, s.y, o);
    }
    return s;
}

// Sums over the threads of a row: one warp, or the block.  Two buffers take
// turns, so one barrier per sum is enough: a thread writes a buffer again
// only after the barrier of the sum in between, which every reader of the
// earlier values has reached.
template <bool WARP>
struct RowSum {
    float2 (*buf)[32];
    int turn = 0;
    __device__ __forceinline__ float2 operator()(float2 s) {
        s = warp_sum(s);
        if (WARP) return s;
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        if (lane == 0) buf[turn][warp] = s;
        __syncthreads();
        s = lane < static_cast<int>(blockDim.x >> 5) ? buf[turn][lane] : make_float2(0.0f, 0.0f);
        turn ^= 1;
        return warp_sum(s);
    }
};

// ------------------------------------------------------------------ rows through shared memory
//
// A ring of slots, each for one row of up to two matrices, filled by bulk
// copies that one thread asks for.  A copy starts and ends on 16-byte
// boundaries, so it may bring up to three floats of the neighbouring rows (or of
// the gap between them) along; a row whose copy would leave the matrix at
// either end is read directly instead.

constexpr int kMaxSlots = 8;

struct RowSource {
    const float* base;
    long long ld;
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}

// Where a row's 16-byte aligned copy begins, how long it is, and whether it stays inside the matrix.
struct RowSpan {
    uintptr_t begin;
    uint32_t bytes, skip;  // skip: floats before the row's first
    bool inside;
};

__device__ __forceinline__ RowSpan row_span(const RowSource& m, long long row, long long rows, int cols) {
    const uintptr_t first = reinterpret_cast<uintptr_t>(m.base + row * m.ld);
    const uintptr_t last = first + static_cast<uintptr_t>(cols) * 4;
    RowSpan s;
    s.begin = first & ~static_cast<uintptr_t>(15);
    s.bytes = static_cast<uint32_t>(((last + 15) & ~static_cast<uintptr_t>(15)) - s.begin);
    s.skip = static_cast<uint32_t>(first - s.begin) / 4;
    s.inside = s.begin >= reinterpret_cast<uintptr_t>(m.base) &&
               s.begin + s.bytes <= reinterpret_cast<uintptr_t>(m.base + (rows - 1) * m.ld + cols);
    return s;
}

__host__ __device__ constexpr int row_slot_bytes(int cols) { return (cols * 4 + 12 + 15) / 16 * 16; }

__device__ __forceinline__ float4 ld_shared_v4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}

template <int MATS>
struct RowRing {
    RowSource mats[MATS];
    uint32_t slots;         // shared addresses
    uint32_t bar0;
    int (*skip)[MATS];      // of each slot: floats before its row's first, or -1 where the row is read directly
    int n, cols;
    long long rows;

    // Asks for `row` into `slot`; one thread.  (What it leaves in `skip` is released by its arrival at the barrier.)
    __device__ __forceinline__ void ask(long long row, int slot) const {
        const uint32_t bar = bar0 + 8 * slot, dst = slots + slot * MATS * row_slot_bytes(cols);
        RowSpan s[MATS];
        uint32_t bytes = 0;
#pragma unroll
        for (int m = 0; m < MATS; ++m) {
            s[m] = row_span(mats[m], row, rows, cols);
            bytes += s[m].inside ? s[m].bytes : 0;
            skip[slot][m] = s[m].inside ? static_cast<int>(s[m].skip) : -1;
        }
        mbar_arrive_expect_tx(bar, bytes);
#pragma unroll
        for (int m = 0; m < MATS; ++m)
            if (s[m].inside)
                bulk_load(dst + m * row_slot_bytes(cols), reinterpret_cast<const void*>(s[m].begin), s[m].bytes, bar);
    }

    // This thread's units of matrix m's row: from its slot or, at the matrix's ends, from where it lies; `past` behind it.
    template <int W, int NV>
    __device__ __forceinline__ void take(float (&v)[NV][W], int m, long long row, int slot, int t, int threads,
                                         float past = 0.0f) const {
        const int ahead = skip[slot][m];
        if (ahead >= 0) {
            const uint32_t at = slots + (slot * MATS + m) * row_slot_bytes(cols) + (ahead + t * W) * 4;
#pragma unroll
            for (int u = 0; u < NV; ++u) {
                const int c = (u * threads + t) * W;
                if (W == 4 && c + W <= cols) {
                    const float4 x = ld_shared_v4(at + u * threads * W * 4);
                    v[u][0] = x.x;
                    v[u][W > 1 ? 1 : 0] = x.y;
                    v[u][W > 2 ? 2 : 0] = x.z;
                    v[u][W > 3 ? 3 : 0] = x.w;
                } else {
#pragma unroll
                    for (int i = 0; i < W; ++i)
                        v[u][i] = W == 1 || c + i < cols ? load_shared_if(c + i < cols, at + (u * threads * W + i) * 4, past) : past;
                }
            }
        } else {
            const float* p = mats[m].base + row * mats[m].ld;
#pragma unroll
            for (int u = 0; u < NV; ++u) load_unit<W>(v[u], p, (u * threads + t) * W, cols, past);
        }
    }
};

constexpr int kWarpRowThreads = 256;  // blocks of eight warps, a row each

struct NormStats {
    float mean, rstd;
};

// Mean and 1 / sqrt(var + eps) of a row that its threads hold in v; `sum` adds over them.
template <int W, int NV, typename Sum>
__device__ __forceinline__ NormStats norm_stats(const float (&v)[NV][W], int t, int threads, const NormParams& p, float inv,
                                                Sum sum) {
    float s = 0.0f;
#pragma unroll
    for (int u = 0; u < NV; ++u)
#pragma unroll
        for (int i = 0; i < W; ++i) s += v[u][i];
    NormStats st;
    st.mean = sum(s) * inv;
    s = 0.0f;
#pragma unroll
    for (int u = 0; u < NV; ++u)
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const float d = (u * threads + t) * W + i < p.cols ? v[u][i] - st.mean : 0.0f;
            s += d * d;
        }
    st.rstd = 1.0f / sqrtf(sum(s) * inv + p.eps);
    return st;
}

// gamma and beta of a thread's columns, in registers: the ring leaves L1 little room, and read again for every row
// they took 16384 x 4096 from 88 to 114 us.  (The warp kernels, whose blocks leave L1 alone, read them from there
// where a lane holds more than 16 columns.)
template <int W, int NV, bool HELD>
struct NormAffine {
    static constexpr bool kHeld = HELD;
    float g[kHeld ? NV : 1][W], b[kHeld ? NV : 1][W];
    __device__ __forceinline__ NormAffine(const NormParams& p, int t, int threads) {
        if constexpr (kHeld) {
#pragma unroll
            for (int u = 0; u < NV; ++u) read(u, u, p, t, threads);
        }
    }
    __device__ __forceinline__ void read(int into, int u, const NormParams& p, int t, int threads) {
        load_param<W, true>(g[into], p.gamma, (u * threads + t) * W, p.cols, 1.0f);
        load_param<W, true>(b[into], p.beta, (u * threads + t) * W, p.cols, 0.0f);
    }
};

template <int W, int NV, bool HELD>
__device__ __forceinline__ void norm_out(float (&v)[NV][W], const NormStats& st, NormAffine<W, NV, HELD>& affine, int t, int threads,
                                         long long row, const NormParams& p) {
    if (t == 0) {
        if (p.mean) p.mean[row] = st.mean;
        if (p.rstd) p.rstd[row] = st.rstd;
    }
    float* y = p.y + row * p.ldy;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
        const int at = HELD ? u : 0;
        if constexpr (!HELD) affine.read(0, u, p, t, threads);
#pragma unroll
        for (int i = 0; i < W; ++i) v[u][i] = (v[u][i] - st.mean) * st.rstd * affine.g[at][i] + affine.b[at][i];
        store_unit<W>(v[u], y, (u * threads + t) * W, p.cols);
    }
}

// Rows of up to 1024 columns, a warp each: lane t holds NV units of W floats, unit u at columns (32 u + t) * W.
template <int W, int NV>
__global__ void __launch_bounds__(kWarpRowThreads) layer_norm_warp_kernel(const NormParams p) {
    const int t = threadIdx.x & 31;
    const long long rows_at_once = static_cast<long long>(gridDim.x) * (kWarpRowThreads / 32);
    const float inv = 1.0f / static_cast<float>(p.cols);
    wait_for_previous_kernel();
    let_next_kernel_in();
    NormAffine<W, NV, W * NV <= 16> affine(p, t, 32);
    for (long long row = blockIdx.x * static_cast<long long>(kWarpRowThreads / 32) + (threadIdx.x >> 5); row < p.rows;
         row += rows_at_once) {
        const float* x = p.x + row * p.ldx;
        float v[NV][W];
#pragma unroll
        for (int u = 0; u < NV; ++u) load_unit<W>(v[u], x, (u * 32 + t) * W, p.cols);
        const NormStats st = norm_stats<W, NV>(v, t, 32, p, inv, [](float s) { return warp_sum(make_float2(s, 0.0f)).x; });
        norm_out(v, st, affine, t, 32, row, p);
    }
}

// Longer rows, a block each.
template <int W, int NV>
__global__ void __launch_bounds__(W * NV > 8 ? 512 : 1024) layer_norm_block_kernel(const NormParams p, int slots) {
    __shared__ float2 buf[2][32];
    __shared__ uint64_t bars[kMaxSlots];
    __shared__ int failed;  // the first round whose copy did not arrive: every thread leaves in that round
    extern __shared__ __align__(16) uint8_t ring_smem[];
    RowSum<false> row_sum{buf};
    __shared__ int skip[kMaxSlots][1];
    const RowRing<1> ring{{{p.x, p.ldx}}, smem_addr(ring_smem), smem_addr(bars), skip, slots, p.cols, p.rows};
    const int threads = blockDim.x, t = threadIdx.x;
    const float inv = 1.0f / static_cast<float>(p.cols);
    if (t == 0) {
        for (int s = 0; s < slots; ++s) mbar_init(ring.bar0 + 8 * s, 1);
        failed = INT_MAX;
        fence_barrier_init();
    }
    wait_for_previous_kernel();
    let_next_kernel_in();
    if (t == 0) {
        for (int s = 0; s < slots; ++s) {
            const long long row = blockIdx.x + static_cast<long long>(s) * gridDim.x;
            if (row < p.rows) ring.ask(row, s);
        }
    }
    __syncthreads();
    NormAffine<W, NV, true> affine(p, t, threads);
    int slot = 0, round = 0;
    uint32_t phase = 0;
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x, ++round) {
        if (!mbar_wait(ring.bar0 + 8 * slot, phase, p.timeout_ns)) atomicMin(&failed, round);
        float v[NV][W];
        ring.take(v, 0, row, slot, t, threads);
        // The first sum's barrier says that every thread has taken its part: the slot can be filled again.
        bool first = true;
        const NormStats st = norm_stats<W, NV>(v, t, threads, p, inv, [&](float s) {
            const float r = row_sum(make_float2(s, 0.0f)).x;
            const long long ahead = row + static_cast<long long>(slots) * gridDim.x;
            if (first && t == 0 && ahead < p.rows && failed > round) ring.ask(ahead, slot);
            first = false;
            return r;
        });
        if (failed <= round) break;
        norm_out(v, st, affine, t, threads, row, p);
        if (++slot == slots) { slot = 0; phase ^= 1u; }
    }
    if (t == 0 && failed != INT_MAX) {
        atomicOr(p.err, kErrProducer);
        for (int s = 0; s < 2 * slots; ++s) mbar_wait(ring.bar0 + 8 * (s % slots), s / slots, p.timeout_ns);
    }
}

// Rows too long for a block's registers: three passes over the row, the
// second and third from L2.
template <int W>
__global__ void __launch_bounds__(1024) layer_norm_long_kernel(const NormParams p) {
    __shared__ float2 buf[2][32];
    RowSum<false> row_sum{buf};
    const int step = blockDim.x * W;
    const float inv = 1.0f / static_cast<float>(p.cols);
    wait_for_previous_kernel();
    let_next_kernel_in();
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const float* x = p.x + row * p.ldx;
        float* y = p.y + row * p.ldy;
        float v[W];
        float2 s = make_float2(0.0f, 0.0f);
        for (long long c = threadIdx.x * W; c < p.cols; c += step) {
            load_unit<W>(v, x, static_cast<int>(c), p.cols);
#pragma unroll
            for (int i = 0; i < W; ++i) s.x += v[i];
        }
        const float mean = row_sum(s).x * inv;
        s = make_float2(0.0f, 0.0f);
        for (long long c = threadIdx.x * W; c < p.cols; c += step) {
            load_unit<W>(v, x, static_cast<int>(c), p.cols);
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const float d = c + i < p.cols ? v[i] - mean : 0.0f;
                s.x += d * d;
            }
        }
        const float rstd = 1.0f / sqrtf(row_sum(s).x * inv + p.eps);
        if (threadIdx.x == 0) {
            if (p.mean) p.mean[row] = mean;
            if (p.rstd) p.rstd[row] = rstd;
        }
        for (long long c = threadIdx.x * W; c < p.cols; c += step) {
            float g[W], b[W];
            load_unit<W>(v, x, static_cast<int>(c), p.cols);
            load_param<W, true>(g, p.gamma, static_cast<int>(c), p.cols, 1.0f);
            load_param<W, true>(b, p.beta, static_cast<int>(c), p.cols, 0.0f);
#pragma unroll
            for (int i = 0; i < W; ++i) v[i] = (v[i] - mean) * rstd * g[i] + b[i];
            store_unit<W>(v, y, static_cast<int>(c), p.cols);
        }
    }
}

// What the forward pass saved of a row.
__device__ __forceinline__ NormStats saved_stats(const NormGradParams& p, long long row) {
    if (row >= p.rows) return {0.0f, 0.0f};
    return {__ldg(p.mean + row), __ldg(p.rstd + row)};
}

// One row of the backward pass, held by `threads` threads: xh and d come in as x and dy, the mean and 0 past the row's end
// (not 0 and 0: a mean times rstd past fp32's range would make the sums NaN there); dx goes out, and the thread's columns
// of dgamma and dbeta grow.
template <int W, int NV, typename Sum>
__device__ __forceinline__ void norm_grad_row(float (&xh)[NV][W], float (&d)[NV][W], float (&dg)[NV][W], float (&db)[NV][W],
                                              const float (&gamma)[NV][W], NormStats st, int t, int threads, long long row, const NormGradParams& p, float inv, Sum sum) {
    const float mean = st.mean, rstd = st.rstd;
    float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int u = 0; u < NV; ++u) {
#pragma unroll
        for (int i = 0; i < W; ++i) {
            // Columns past the row have xh = d = 0: they add nothing to any sum.
            xh[u][i] = (xh[u][i] - mean) * rstd;
            dg[u][i] += d[u][i] * xh[u][i];
            db[u][i] += d[u][i];
            d[u][i] *= gamma[u][i];
            s.x += d[u][i];
            s.y += d[u][i] * xh[u][i];
        }
    }
    s = sum(s);
    if (!p.dx) return;
    const float m1 = s.x * inv, m2 = s.y * inv;
    float* dx = p.dx + row * p.lddx;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
#pragma unroll
        for (int i = 0; i < W; ++i) d[u][i] = rstd * (d[u][i] - m1 - xh[u][i] * m2);
        store_unit<W>(d[u], dx, (u * threads + t) * W, p.cols);
    }
}

template <int W, int NV>
__global__ void __launch_bounds__(kWarpRowThreads) layer_norm_grad_warp_kernel(const NormGradParams p) {
    extern __shared__ __align__(16) uint8_t smem[];
    float* block_acc = reinterpret_cast<float*>(smem);  // [2][cols]: the block's sums over its warps
    constexpr int threads = 32;
    const int t = threadIdx.x & 31;
    const long long rows_at_once = static_cast<long long>(gridDim.x) * (kWarpRowThreads / 32);
    const float inv = 1.0f / static_cast<float>(p.cols);
    float dg[NV][W] = {}, db[NV][W] = {}, gamma[NV][W];
#pragma unroll
    for (int u = 0; u < NV; ++u) load_param<W, false>(gamma[u], p.gamma, (u * threads + t) * W, p.cols, 1.0f);
    long long row = blockIdx.x * static_cast<long long>(kWarpRowThreads / 32) + (threadIdx.x >> 5);
    NormStats next = saved_stats(p, row);  // a row ahead, so that no row waits for its two numbers
    for (; row < p.rows; row += rows_at_once) {
        const NormStats st = next;
        next = saved_stats(p, row + rows_at_once);
        float xh[NV][W], d[NV][W];
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            load_unit<W>(xh[u], p.x + row * p.ldx, (u * 32 + t) * W, p.cols, st.mean);
            load_unit<W>(d[u], p.dy + row * p.lddy, (u * 32 + t) * W, p.cols);
        }
        norm_grad_row<W, NV>(xh, d, dg, db, gamma, st, t, 32, row, p, inv, [](float2 s) { return warp_sum(s); });
    }
    if (!p.partial) return;
    // The warps add their sums one after the other, in warp order.
    for (int w = 0; w < kWarpRowThreads / 32; ++w) {
        if (static_cast<int>(threadIdx.x >> 5) == w) {
#pragma unroll
            for (int u = 0; u < NV; ++u)
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    const int c = (u * 32 + t) * W + i;
                    if (c < p.cols) {
                        block_acc[c] = (w ? block_acc[c] : 0.0f) + dg[u][i];
                        block_acc[p.cols + c] = (w ? block_acc[p.cols + c] : 0.0f) + db[u][i];
                    }
                }
        }
        __syncthreads();
    }
    float* out = p.partial + static_cast<long long>(blockIdx.x) * 2 * p.cols;
    for (int c = threadIdx.x; c < 2 * p.cols; c += kWarpRowThreads) out[c] = block_acc[c];
}

template <int W, int NV>
__global__ void __launch_bounds__(W * NV > 8 ? 512 : 1024) layer_norm_grad_block_kernel(const NormGradParams p, int slots) {
    __shared__ float2 buf[2][32];
    __shared__ uint64_t bars[kMaxSlots];
    __shared__ int failed;  // the first round whose copy did not arrive: every thread leaves in that round
    extern __shared__ __align__(16) uint8_t smem[];
    RowSum<false> row_sum{buf};
    __shared__ int skip[kMaxSlots][2];
    const RowRing<2> ring{{{p.x, p.ldx}, {p.dy, p.lddy}}, smem_addr(smem), smem_addr(bars), skip, slots, p.cols, p.rows};
    const int threads = blockDim.x, t = threadIdx.x;
    const float inv = 1.0f / static_cast<float>(p.cols);
    if (t == 0) {
        for (int s = 0; s < slots; ++s) mbar_init(ring.bar0 + 8 * s, 1);
        failed = INT_MAX;
        fence_barrier_init();
        for (int s = 0; s < slots; ++s) {
            const long long row = blockIdx.x + static_cast<long long>(s) * gridDim.x;
            if (row < p.rows) ring.ask(row, s);
        }
    }
    __syncthreads();
    float dg[NV][W] = {}, db[NV][W] = {}, gamma[NV][W];
#pragma unroll
    for (int u = 0; u < NV; ++u) load_param<W, false>(gamma[u], p.gamma, (u * threads + t) * W, p.cols, 1.0f);
    int slot = 0, round = 0;
    uint32_t phase = 0;
    NormStats next = saved_stats(p, blockIdx.x);  // a row ahead, so that no row waits for its two numbers
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x, ++round) {
        const NormStats st = next;
        next = saved_stats(p, row + gridDim.x);
        if (!mbar_wait(ring.bar0 + 8 * slot, phase, p.timeout_ns)) atomicMin(&failed, round);
        float xh[NV][W], d[NV][W];
        ring.take(d, 1, row, slot, t, threads);
        ring.take(xh, 0, row, slot, t, threads, st.mean);
        // The sum's barrier says that every thread has taken its part: the slot can be filled again.
        norm_grad_row<W, NV>(xh, d, dg, db, gamma, st, t, threads, row, p, inv, [&](float2 s) {
            s = row_sum(s);
            const long long ahead = row + static_cast<long long>(slots) * gridDim.x;
            if (t == 0 && ahead < p.rows && failed > round) ring.ask(ahead, slot);
            return s;
        });
        if (failed <= round) break;
        if (++slot == slots) { slot = 0; phase ^= 1u; }
    }
    if (t == 0 && failed != INT_MAX) {
        atomicOr(p.err, kErrProducer);
        for (int s = 0; s < 2 * slots; ++s) mbar_wait(ring.bar0 + 8 * (s % slots), s / slots, p.timeout_ns);
    }
    if (!p.partial) return;
    float* out = p.partial + static_cast<long long>(blockIdx.x) * 2 * p.cols;
#pragma unroll
    for (int u = 0; u < NV; ++u)
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const int c = (u * threads + t) * W + i;
            if (c < p.cols) {
                out[c] = dg[u][i];
                out[p.cols + c] = db[u][i];
            }
        }
}

// Rows of up to 16384 columns: x and dy in the registers of 1024 threads, the sums for dgamma and dbeta, for
// which none are left, in shared memory, each column touched by one thread only.
template <int W>
__global__ void __launch_bounds__(1024) layer_norm_grad_wide_kernel(const NormGradParams p) {
    constexpr int NV = 16 / W;
    __shared__ float2 buf[2][32];
    extern __shared__ __align__(16) uint8_t smem[];
    float* acc = reinterpret_cast<float*>(smem);  // [2][cols]
    RowSum<false> row_sum{buf};
    const int t = threadIdx.x;
    const float inv = 1.0f / static_cast<float>(p.cols);
    for (int c = t; c < 2 * p.cols; c += 1024) acc[c] = 0.0f;
    __syncthreads();
    NormStats next = saved_stats(p, blockIdx.x);
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const NormStats st = next;
        next = saved_stats(p, row + gridDim.x);
        float xh[NV][W], d[NV][W];
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            load_unit<W>(xh[u], p.x + row * p.ldx, (u * 1024 + t) * W, p.cols, st.mean);
            load_unit<W>(d[u], p.dy + row * p.lddy, (u * 1024 + t) * W, p.cols);
        }
        float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            float g[W];
            load_param<W, false>(g, p.gamma, (u * 1024 + t) * W, p.cols, 1.0f);
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const int c = (u * 1024 + t) * W + i;
                xh[u][i] = (xh[u][i] - st.mean) * st.rstd;
                if (c < p.cols) {
                    acc[c] += d[u][i] * xh[u][i];
                    acc[p.cols + c] += d[u][i];
                }
                d[u][i] *= g[i];
                s.x += d[u][i];
                s.y += d[u][i] * xh[u][i];
            }
        }
        if (!p.dx) continue;
        s = row_sum(s);
        const float m1 = s.x * inv, m2 = s.y * inv;
#pragma unroll
        for (int u = 0; u < NV; ++u) {
#pragma unroll
            for (int i = 0; i < W; ++i) d[u][i] = st.rstd * (d[u][i] - m1 - xh[u][i] * m2);
            store_unit<W>(d[u], p.dx + row * p.lddx, (u * 1024 + t) * W, p.cols);
        }
    }
    if (!p.partial) return;
    float* out = p.partial + static_cast<long long>(blockIdx.x) * 2 * p.cols;
    __syncthreads();
    for (int c = t; c < 2 * p.cols; c += 1024) out[c] = acc[c];
}

// Rows too long for a block's registers: x and dy are read twice, and the
// block's partial sums live in its own row of the workspace, each column
// touched by one thread only.
template <int W>
__global__ void __launch_bounds__(1024) layer_norm_grad_long_kernel(const NormGradParams p) {
    __shared__ float2 buf[2][32];
    RowSum<false> row_sum{buf};
    const int step = blockDim.x * W;
    const float inv = 1.0f / static_cast<float>(p.cols);
    float* acc = p.partial ? p.partial + static_cast<long long>(blockIdx.x) * 2 * p.cols : nullptr;
    bool first = true;
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const float mean = __ldg(p.mean + row), rstd = __ldg(p.rstd + row);
        const float* x = p.x + row * p.ldx;
        const float* dy = p.dy + row * p.lddy;
        float xh[W], d[W], g[W];
        float2 s = make_float2(0.0f, 0.0f);
        for (long long cc = threadIdx.x * W; cc < p.cols; cc += step) {
            const int c = static_cast<int>(cc);
            load_unit<W>(xh, x, c, p.cols, mean);
            load_unit<W>(d, dy, c, p.cols);
            load_param<W, false>(g, p.gamma, c, p.cols, 1.0f);
#pragma unroll
            for (int i = 0; i < W; ++i) {
                xh[i] = (xh[i] - mean) * rstd;
                if (acc && c + i < p.cols) {
                    acc[c + i] = (first ? 0.0f : acc[c + i]) + d[i] * xh[i];
                    acc[p.cols + c + i] = (first ? 0.0f : acc[p.cols + c + i]) + d[i];
                }
                s.x += d[i] * g[i];
                s.y += d[i] * g[i] * xh[i];
            }
        }
        first = false;
        if (!p.dx) continue;
        s = row_sum(s);
        const float m1 = s.x * inv, m2 = s.y * inv;
        float* dx = p.dx + row * p.lddx;
        for (long long cc = threadIdx.x * W; cc < p.cols; cc += step) {
            const int c = static_cast<int>(cc);
            load_unit<W>(xh, x, c, p.cols, mean);
            load_unit<W>(d, dy, c, p.cols);
            load_param<W, false>(g, p.gamma, c, p.cols, 1.0f);
#pragma unroll
            for (int i = 0; i < W; ++i) {
                xh[i] = (xh[i] - mean) * rstd;
                d[i] = rstd * (d[i] * g[i] - m1 - xh[i] * m2);
            }
            store_unit<W>(d, dx, c, p.cols);
        }
    }
}

// dgamma[c] (blockIdx.y 0) or dbeta[c] (1): the blocks' partial rows, summed by ROWS threads per column and then in
// thread order.  Launched while the backward kernel still runs (its launch latency hides there).
template <int ROWS>
__global__ void __launch_bounds__(32 * ROWS) sum_partials_kernel(const float* partial, int blocks, int cols, float* dgamma,
                                                                 float* dbeta) {
    __shared__ float part[ROWS][33];
    float* out = blockIdx.y ? dbeta : dgamma;
    const int c = blockIdx.x * 32 + threadIdx.x;
    wait_for_previous_kernel();
    if (!out) return;
    float s = 0.0f;
    if (c < cols) {
        const float* src = partial + static_cast<long long>(blockIdx.y) * cols + c;
#pragma unroll 8
        for (int b = threadIdx.y; b < blocks; b += ROWS) s += __ldcg(src + static_cast<long long>(b) * 2 * cols);
    }
    part[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y == 0 && c < cols) {
#pragma unroll
        for (int i = 1; i < ROWS; ++i) s += part[i][threadIdx.x];
        out[c] = s;
    }
}

constexpr int kBlockThreads = 512;                      // of a block that holds more than kWideFloats of a row a thread
constexpr int kWideThreads = 1024, kWideFloats = 8;

// How a row is spread: `threads` threads (32: a warp, eight rows to a block)
// holding `units` units each; units == 0: the kernel for long rows.
struct RowPlan {
    int threads, units;
    bool warp;
};

// warp_floats, block_floats: what a thread may hold of one row.
RowPlan plan_row(int cols, int width, long long rows, int num_sms, int warp_floats, int block_floats) {
    const int total = (cols + width - 1) / width;
    // Few rows leave most SMs without one: the widest block shortens each thread's share of a row.
    const bool few = rows <= 2ll * num_sms;
    if (total <= 32 || (!few && total * width <= 32 * warp_floats)) {
        int units = 1;
        while (32 * units < total) units *= 2;
        return {32, units, true};
    }
    auto threads_for = [&](int units) { return ((total + units - 1) / units + 31) / 32 * 32; };
    if (few) {
        for (int units = 1; units * width <= kWideFloats; units *= 2)
            if (threads_for(units) <= kWideThreads) return {threads_for(units), units, false};
    }
    // Else the smallest block, for many rows side by side on an SM (65536 x 1024 backward: 139 us with 64 threads, 222
    // with 256), unless whole warps of it would idle; 16 floats before more.
    for (int floats = std::min(16, block_floats); floats <= block_floats; floats *= 2) {
        for (int units = floats / width; units >= 1; units /= 2) {
            const int threads = threads_for(units);
            if (threads <= kBlockThreads && 4ll * threads * units <= 5ll * total + 128) return {threads, units, false};
        }
        for (int units = floats / width; units >= 1; units /= 2)
            if (threads_for(units) <= kBlockThreads) return {threads_for(units), units, false};
    }
    return {kWideThreads, 0, false};
}

// Blocks of `threads` threads and `smem` bytes of shared memory that fit on an SM: by the kernel's registers (each of
// the four partitions has 16384, a warp takes 32 times a thread's), the threads and the shared memory.  Computed here,
// because asking the runtime for it takes longer than a small call.
template <auto kernel>
int blocks_per_sm(int threads, size_t smem) {
    static const int regs = [] {
        cudaFuncAttributes a;
        if (cudaFuncGetAttributes(&a, kernel) != cudaSuccess) {
            cudaGetLastError();
            return 255;
        }
        return (a.numRegs + 7) / 8 * 8;
    }();
    const int by_regs = 4 * (16384 / (32 * regs)) / (threads / 32);
    const int by_smem = static_cast<int>(227 * 1024 / (smem + 2048));
    return std::max(1, std::min(std::min(by_regs, 2048 / threads), std::min(by_smem, 32)));
}

// Slots of a ring with `mats` rows to a slot, for a kernel of which `blocks` fit on an SM by their registers: what
// shared memory gives each of them, two at least.
int ring_slots(int blocks, int cols, int mats) {
    return std::max(2, std::min(kMaxSlots, 216 * 1024 / std::min(blocks, 16) / (mats * row_slot_bytes(cols))));
}

constexpr int kRingBytes = 224 * 1024;  // of shared memory that a ring may take, or the wide kernel's sums

constexpr int kNormFloats = 32;      // of a row per thread: 1024 columns per warp, 16384 per block
constexpr int kNormGradFloats = 16;  // x, dy and two sums for each: 512 columns per warp, 8192 per block

template <int W, int NV>
cudaError_t launch_norm(const NormParams& p, const RowPlan& plan, int num_sms, cudaStream_t stream) {
    if (plan.warp) {
        const long long want = (p.rows + kWarpRowThreads / 32 - 1) / (kWarpRowThreads / 32);
        const int blocks = static_cast<int>(
            std::min<long long>(want, static_cast<long long>(num_sms) * blocks_per_sm<layer_norm_warp_kernel<W, NV>>(kWarpRowThreads, 0)));
        return launch_early(layer_norm_warp_kernel<W, NV>, dim3(blocks), dim3(kWarpRowThreads), 0, stream, 1, p);
    } else {
        const cudaError_t e = allow_shared<layer_norm_block_kernel<W, NV>>(kRingBytes);
        if (e != cudaSuccess) return e;
        const int slots = ring_slots(blocks_per_sm<layer_norm_block_kernel<W, NV>>(plan.threads, 0), p.cols, 1);
        const size_t smem = static_cast<size_t>(slots) * row_slot_bytes(p.cols);
        const int blocks = static_cast<int>(
            std::min<long long>(p.rows, static_cast<long long>(num_sms) * blocks_per_sm<layer_norm_block_kernel<W, NV>>(plan.threads, smem)));
        return launch_early(layer_norm_block_kernel<W, NV>, dim3(blocks), dim3(plan.threads), smem, stream, 1, p, slots);
    }
}

template <int W>
cudaError_t launch_norm_width(const NormParams& p, int num_sms, cudaStream_t stream) {
    const RowPlan plan = plan_row(p.cols, W, p.rows, num_sms, kNormFloats, kNormFloats);
    switch (plan.units) {
        case 1: return launch_norm<W, 1>(p, plan, num_sms, stream);
        case 2: return launch_norm<W, 2>(p, plan, num_sms, stream);
        case 4: return launch_norm<W, 4>(p, plan, num_sms, stream);
        case 8: return launch_norm<W, 8>(p, plan, num_sms, stream);
        case 16: return launch_norm<W, W == 1 ? 16 : 8>(p, plan, num_sms, stream);
        case 32: return launch_norm<W, W == 1 ? 32 : 8>(p, plan, num_sms, stream);
        default: break;
    }
    const int blocks = static_cast<int>(
        std::min<long long>(p.rows, static_cast<long long>(num_sms) * blocks_per_sm<layer_norm_long_kernel<W>>(plan.threads, 0)));
    return launch_early(layer_norm_long_kernel<W>, dim3(blocks), dim3(plan.threads), 0, stream, 1, p);
}

// One launch of the backward kernel, or (p == nullptr) the number of blocks it takes.
template <int W, int NV>
cudaError_t launch_norm_grad(const NormGradParams* p, const RowPlan& plan, long long rows, int cols, int num_sms,
                             int* blocks, cudaStream_t stream) {
    if (plan.warp) {
        const size_t smem = 2 * sizeof(float) * cols;
        if (!p) {
            const long long want = (rows + kWarpRowThreads / 32 - 1) / (kWarpRowThreads / 32);
            *blocks = static_cast<int>(
                std::min<long long>(want, static_cast<long long>(num_sms) * blocks_per_sm<layer_norm_grad_warp_kernel<W, NV>>(kWarpRowThreads, smem)));
            return cudaSuccess;
        }
        layer_norm_grad_warp_kernel<W, NV><<<*blocks, kWarpRowThreads, smem, stream>>>(*p);
    } else {
        const int slots = ring_slots(blocks_per_sm<layer_norm_grad_block_kernel<W, NV>>(plan.threads, 0), cols, 2);
        const size_t smem = static_cast<size_t>(slots) * 2 * row_slot_bytes(cols);
        if (!p) {
            const cudaError_t e = allow_shared<layer_norm_grad_block_kernel<W, NV>>(kRingBytes);
            if (e != cudaSuccess) return e;
            *blocks = static_cast<int>(
                std::min<long long>(rows, static_cast<long long>(num_sms) * blocks_per_sm<layer_norm_grad_block_kernel<W, NV>>(plan.threads, smem)));
            return cudaSuccess;
        }
        layer_norm_grad_block_kernel<W, NV><<<*blocks, plan.threads, smem, stream>>>(*p, slots);
    }
    note_launch();
    return cudaGetLastError();
}

template <int W>
cudaError_t launch_norm_grad_width(const NormGradParams* p, long long rows, int cols, int num_sms, int* blocks,
                                   cudaStream_t stream) {
    const RowPlan plan = plan_row(cols, W, rows, num_sms, kNormGradFloats, kNormGradFloats);
    switch (plan.units) {
        case 1: return launch_norm_grad<W, 1>(p, plan, rows, cols, num_sms, blocks, stream);
        case 2: return launch_norm_grad<W, 2>(p, plan, rows, cols, num_sms, blocks, stream);
        case 4: return launch_norm_grad<W, 4>(p, plan, rows, cols, num_sms, blocks, stream);
        case 8: return launch_norm_grad<W, W == 1 ? 8 : 4>(p, plan, rows, cols, num_sms, blocks, stream);
        case 16: return launch_norm_grad<W, W == 1 ? 16 : 4>(p, plan, rows, cols, num_sms, blocks, stream);
        default: break;
    }
    if (cols <= 16 * 1024) {
        const size_t smem = 2 * sizeof(float) * cols;
        if (!p) {
            const cudaError_t e = allow_shared<layer_norm_grad_wide_kernel<W>>(kRingBytes);
            if (e != cudaSuccess) return e;
            *blocks = static_cast<int>(
                std::min<long long>(rows, static_cast<long long>(num_sms) * blocks_per_sm<layer_norm_grad_wide_kernel<W>>(kWideThreads, smem)));
            return cudaSuccess;
        }
        layer_norm_grad_wide_kernel<W><<<*blocks, kWideThreads, smem, stream>>>(*p);
        note_launch();
        return cudaGetLastError();
    }
    if (!p) {
        *blocks = static_cast<int>(
            std::min<long long>(rows, static_cast<long long>(num_sms) * blocks_per_sm<layer_norm_grad_long_kernel<W>>(plan.threads, 0)));
        return cudaSuccess;
    }
    layer_norm_grad_long_kernel<W><<<*blocks, plan.threads, 0, stream>>>(*p);
    note_launch();
    return cudaGetLastError();
}

int layer_norm(GpuCtx* ctx, NormParams p, void* stream) {
    if (!ctx || p.rows < 0 || p.cols < 1 || p.ldx < p.cols || p.ldy < p.cols || (p.rows > 0 && (!p.x || !p.y))) {
        set_error("mxb_layer_norm: invalid arguments");
        return MXB_E_ARG;
    }
    if (p.x == p.y && p.ldx != p.ldy) {
        set_error("mxb_layer_norm: in place, x and y need the same pitch");
        return MXB_E_ARG;
    }
    if (p.cols > kMaxExtent) {
        set_error("mxb_layer_norm: cols is limited to 2^30");
        return MXB_E_UNSUPPORTED;
    }
    if (p.rows == 0) return MXB_OK;
    DeviceScope scope(ctx->device);
    cudaStream_t st = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
    const bool vec = aligned16(p.x) && aligned16(p.y) && aligned16(p.gamma) && aligned16(p.beta) && p.ldx % 4 == 0 &&
                     p.ldy % 4 == 0;
    p.timeout_ns = ctx->timeout_ns;
    p.err = ctx->d_err;
    const cudaError_t e = vec ? launch_norm_width<4>(p, ctx->num_sms, st) : launch_norm_width<1>(p, ctx->num_sms, st);
    return cuda_ok(e, "layer norm launch") ? MXB_OK : MXB_E_CUDA;
}

int layer_norm_backward(GpuCtx* ctx, NormGradParams p, float* dgamma, float* dbeta, void* stream) {
    if (!ctx || p.rows < 0 || p.cols < 1 || p.lddy < p.cols || p.ldx < p.cols || (p.dx && p.lddx < p.cols) ||
        (!p.dx && !dgamma && !dbeta) || (p.rows > 0 && (!p.dy || !p.x || !p.mean || !p.rstd))) {
        set_error("mxb_layer_norm_backward: invalid arguments");
        return MXB_E_ARG;
    }
    if ((p.dx == p.dy && p.lddx != p.lddy) || (p.dx == p.x && p.lddx != p.ldx)) {
        if (p.dx) {
            set_error("mxb_layer_norm_backward: in place, dx needs the pitch of the matrix that it replaces");
            return MXB_E_ARG;
        }
    }
    if (p.cols > kMaxExtent) {
        set_error("mxb_layer_norm_backward: cols is limited to 2^30");
        return MXB_E_UNSUPPORTED;
    }
    DeviceScope scope(ctx->device);
    cudaStream_t st = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
    if (p.rows == 0) {
        for (float* z : {dgamma, dbeta})
            if (z && !cuda_ok(cudaMemsetAsync(z, 0, sizeof(float) * p.cols, st), "layer norm gradient clear"))
                return MXB_E_CUDA;
        return MXB_OK;
    }
    const bool vec = aligned16(p.x) && aligned16(p.dy) && aligned16(p.dx) && aligned16(p.gamma) && p.ldx % 4 == 0 &&
                     p.lddy % 4 == 0 && (!p.dx || p.lddx % 4 == 0);
    auto run = [&](const NormGradParams* q, int* blocks) {
        return vec ? launch_norm_grad_width<4>(q, p.rows, p.cols, ctx->num_sms, blocks, st)
                   : launch_norm_grad_width<1>(q, p.rows, p.cols, ctx->num_sms, blocks, st);
    };
    p.timeout_ns = ctx->timeout_ns;
    p.err = ctx->d_err;
    int blocks = 0;
    if (!cuda_ok(run(nullptr, &blocks), "layer norm backward plan")) return MXB_E_CUDA;
    Scratch scratch(ctx, st);
    if (dgamma || dbeta) {
        p.partial = static_cast<float*>(scratch.alloc(sizeof(float) * 2 * p.cols * static_cast<size_t>(blocks)));
        if (!p.partial) return MXB_E_NOMEM;
    }
    if (!cuda_ok(run(&p, &blocks), "layer norm backward launch")) return MXB_E_CUDA;
    if (!p.partial) return MXB_OK;
    // Many columns fill the SMs with small blocks; few columns need more threads for each.
    const bool tall = p.cols <= 32 * ctx->num_sms;
    const cudaError_t e = launch_early(tall ? sum_partials_kernel<32> : sum_partials_kernel<8>, dim3((p.cols + 31) / 32, 2),
                                       dim3(32, tall ? 32 : 8), 0, st, 1, p.partial, blocks, p.cols, dgamma, dbeta);
    return cuda_ok(e, "layer norm gradient sums launch") ? MXB_OK : MXB_E_CUDA;
}

}  // namespace
}  // namespace mxb

extern "C" {

int mxb_layer_norm(GpuCtx* ctx, const float* x, long long ldx, const float* gamma, const float* beta, float eps,
                   float* y, long long ldy, float* mean, float* rstd, long long rows, int cols, void* stream) {
    try {
        return mxb::layer_norm(ctx, mxb::NormParams{x, ldx, gamma, beta, eps, y, ldy, mean, rstd, rows, cols, 0, nullptr},
                               stream);
    } catch (const std::exception& e) {  // a lock that cannot be taken
        mxb::set_error("mxb_layer_norm: %s", e.what());
        return MXB_E_CUDA;
    }
}

int mxb_layer_norm_backward(GpuCtx* ctx, const float* dy, long long lddy, const float* x, long long ldx,
                            const float* gamma, const float* mean, const float* rstd, float* dx, long long lddx,
                            float* dgamma, float* dbeta, long long rows, int cols, void* stream) {
    try {
        return mxb::layer_norm_backward(
            ctx, mxb::NormGradParams{dy, lddy, x, ldx, gamma, mean, rstd, dx, lddx, nullptr, rows, cols, 0, nullptr}, dgamma,
            dbeta, stream);
    } catch (const std::exception& e) {  // host allocations of the pool's lists
        mxb::set_error("mxb_layer_norm_backward: %s", e.what());
        return MXB_E_NOMEM;
    }
}

}  // extern "C"
