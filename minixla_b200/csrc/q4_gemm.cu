// Products with 4-bit weights and group scales (mxb_q4_gemm):
//   out[m, n] = epi(sum over groups g of s[n, g] * sum over k in g of A[m, k] * (q[n, k] - z[n, g])).
#include "gemm_common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <exception>
#include <mutex>

#include "epilogue_cell.cuh"
#include "runtime_internal.h"

namespace mxb {

namespace {

struct Q4Params {
    const float* a;
    long long lda;
    const unsigned char* q;
    long long ldq;
    const void* scales;
    const unsigned char* zeros;
    long long lds;
    int scale_type, group;
    float* out;
    long long ldo;
    int M, N, K;
    unsigned long long timeout_ns;
    int* err;
    CellEpilogue epi;
};

// ---------------------------------------------------------------- few rows
//
// Up to 16 rows: bound by the weights' bytes.  One mma.sync.m16n8k16 (bf16,
// fp32 accumulate) takes 16 weight columns as its rows and activations as
// its eight columns.  q - z is exact in bf16; an activation is cut into three
// bf16 parts of eight bits each whose sum is exact, so nothing is rounded
// before the fp32 sums.  A warp takes every eighth run of k for
// 16 * MT weight columns; lane (g, t) of the warp holds, for each 32 k, the
// eight values of word t of weight rows g and g + 8 -- the k order inside an
// MMA is free as long as weights and activations agree on it, so the words
// are used as they lie -- and the same eight k of activation row g, which it
// cuts itself.  All 16 k of an MMA lie in one group; the sums of a group (of
// at most a run of it) start from zero and are scaled in fp32.
//  PACK: one or two rows (that many); the eight MMA columns hold the parts
//        side by side (column 3 m + part), one MMA instead of three, and the
//        warp cuts its run once instead of every lane its own eight values.
//  RT:   row tiles of eight; their three parts go through three MMAs into
//        the same accumulators.
// Each warp has a ring of its own: one lane asks TMA for the next run's
// weights and activations (zeros past their edges), so that no instruction
// is spent on addresses and bounds.

constexpr int kFewWarps = 8;

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Two q - z as a bf16 pair, from nibbles 0 and 4 of `w` and the pair (128 + z, 128 + z):
// 0x4300 | q is the bf16 number 128 + q, and the difference is exact.
__device__ __forceinline__ uint32_t weight_pair(uint32_t w, uint32_t z128) {
    uint32_t v;
    asm("lop3.b32 %0, %1, 0x000F000F, %2, 0xEA;" : "=r"(v) : "r"(w), "r"(0x43004300u));  // (w & mask) | magic
    const __nv_bfloat162 h =
        __hsub2(*reinterpret_cast<__nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&z128));
    return *reinterpret_cast<const uint32_t*>(&h);
}

// The top eight bits of x and y as a bf16 pair; x and y keep the rest.
__device__ __forceinline__ uint32_t cut_pair(float& x, float& y) {
    const uint32_t ux = __float_as_uint(x), uy = __float_as_uint(y);
    x -= __uint_as_float(ux & 0xFFFF0000u);
    y -= __uint_as_float(uy & 0xFFFF0000u);
    return __byte_perm(ux, uy, 0x7632);
}

template <int PACK, int RT, int MT, int SHIFT>
struct FewCfg {
    static constexpr int kRows = PACK ? PACK : 8 * RT;
    // k of one unit: 128 bytes of a weight row, or 64 where eight or more rows of activations come with them.
    static constexpr int kRun = PACK ? 256 : 128;
    static constexpr int kPieces = kRun / 32;                       // of 32 k
    static constexpr int kWeightBytes = 16 * MT * kRun / 2;
    static constexpr int kPieceBytes = kRows * 128;                 // 32 k of each row
    static constexpr int kUnit = kWeightBytes + kPieces * kPieceBytes;  // a multiple of 1 KiB
    static constexpr int kStretches = kPieces >> SHIFT;             // of a run, each in one group
    static constexpr int kScaleBytes = (16 * MT + 8) * kStretches * 8;  // per warp: (scale, zero pair) [stretch][row]
    static constexpr int kPartBytes = PACK * kPieces * 3 * 4 * 16;  // per warp: [piece][MMA column][lane t]
    static constexpr int kWarpExtra = kScaleBytes + kPartBytes;
    // As many units as fit in half the shared memory (two CTAs), or in all of it.
    static constexpr int kHalf = (111 * 1024 / kFewWarps - kWarpExtra) / kUnit;
    static constexpr int kAll = (220 * 1024 / kFewWarps - kWarpExtra) / kUnit;
    static constexpr int kDepth = kHalf >= 2 ? (kHalf > 4 ? 4 : kHalf) : (kAll > 4 ? 4 : kAll);
    static constexpr int kRing = kUnit * kFewWarps * kDepth;
    static constexpr int kExtraOffset = kRing;
    static constexpr int kBarOffset = kExtraOffset + kFewWarps * kWarpExtra;
    static constexpr int kReduce = kFewWarps * 16 * MT * (8 * RT) * 4;
    static constexpr int kSmem = 1024 + kBarOffset + kFewWarps * kDepth * 8 + 16;
    static_assert(kUnit % 1024 == 0 && kDepth >= 2 && kReduce <= kRing && kSmem <= 227 * 1024, "shared memory layout");
};

template <int PACK, int RT, int MT, int SHIFT>
__global__ void __launch_bounds__(32 * kFewWarps)
    q4_few_rows_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_a,
                       const __grid_constant__ Q4Params p) {
    using C = FewCfg<PACK, RT, MT, SHIFT>;
    constexpr int kRun = C::kRun, kPieces = C::kPieces;
    extern __shared__ uint8_t smem_raw[];
    // (an offset, not a rounded pointer: the compiler then still knows that these are shared addresses)
    uint8_t* smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * 16 * MT, m0 = blockIdx.y * C::kRows;
    const int rows = min(C::kRows, p.M - m0);
    const int runs = (p.K + kRun - 1) / kRun;
    uint8_t* ring = smem + warp * C::kDepth * C::kUnit;
    uint8_t* extra = smem + C::kExtraOffset + warp * C::kWarpExtra;
    const uint32_t bar0 = smem_addr(smem + C::kBarOffset) + warp * C::kDepth * 8;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::kBarOffset + kFewWarps * C::kDepth * 8);
    if (lane == 0) {
        for (int d = 0; d < C::kDepth; ++d) mbar_init(bar0 + 8 * d, 1);
        fence_barrier_init();
    }
    if (threadIdx.x == 0) *abort_flag = 0;
    __syncthreads();

    // Unit of run r into slot `slot`.  Weights: row i's 16-byte chunk c (piece c, 32 k) at c ^ (i & 7), or at
    // c ^ ((i >> 1) & 3) in a row of 64 bytes; activations: a box for each piece, row m's 128 bytes at 128 m,
    // chunk c at c ^ (m & 7) (the copies' swizzles, conflict-free for the reads below), or (PACK) row by row.
    auto issue = [&](int r, int slot) {
        const uint32_t dst = smem_addr(ring + slot * C::kUnit), bar = bar0 + 8 * slot;
        mbar_arrive_expect_tx(bar, C::kUnit);
        tma_load_2d(dst, &tm_w, bar, r * (kRun / 2), n0);
#pragma unroll
        for (int c = 0; c < (PACK ? 1 : kPieces); ++c)
            tma_load_2d(dst + C::kWeightBytes + c * C::kPieceBytes, &tm_a, bar, r * kRun + 32 * c, m0);
    };
    // The run's scales and zero points, one for each weight row and stretch, spread over the lanes
    // (neighbouring lanes take neighbouring stretches of a row) and loaded a run ahead, unconverted, so that
    // nothing waits for them here.
    constexpr int kEntries = 16 * MT * C::kStretches, kOwn = (kEntries + 31) / 32;
    uint32_t s_raw[kOwn], z_raw[kOwn];
    auto load_group = [&](int r) {
        const int k = r * kRun + (lane % C::kStretches << SHIFT) * 32;
        const long long piece = k / p.group;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            const int row = (32 * i + lane) / C::kStretches, n = n0 + row;
            s_raw[i] = 0;
            z_raw[i] = 8;
            if (row < 16 * MT && n < p.N && k < p.K) {
                const long long at = n * p.lds + piece;
                s_raw[i] = p.scale_type == MXB_SCALE_F32 ? __ldg(static_cast<const uint32_t*>(p.scales) + at)
                                                         : __ldg(static_cast<const unsigned short*>(p.scales) + at);
                if (p.zeros) z_raw[i] = __ldg(p.zeros + at);
            }
        }
    };

    // What this lane reads, as offsets into a unit, the scales and the parts.
    int w_at[kPieces];
#pragma unroll
    for (int c = 0; c < kPieces; ++c)
        w_at[c] = g * (kRun / 2) + ((c ^ (kPieces == 8 ? g : g >> 1)) << 4) + 4 * t;
    const uint2* scale_at = reinterpret_cast<const uint2*>(extra) + g;

    const int part_at = min(g, 3 * PACK - 1) * 4 + t;  // (columns without a part repeat the last: not stored)
    float tot[MT][RT][4] = {};
    int r = warp;
    if (lane == 0) {
#pragma unroll
        for (int d = 0; d < C::kDepth - 1; ++d)
            if (r + d * kFewWarps < runs) issue(r + d * kFewWarps, d);
    }
    if (r < runs) load_group(r);
    uint32_t phase = 0;
    bool failed = false;
    for (int slot = 0; r < runs; r += kFewWarps) {
        __syncwarp();  // the unit, scales and parts before these are read by every lane
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            const int e = 32 * i + lane;
            const uint32_t raw = s_raw[i], z = z_raw[i] & 15u;
            const uint32_t sc = p.scale_type == MXB_SCALE_F32   ? raw
                                : p.scale_type == MXB_SCALE_F16 ? __float_as_uint(__half2float(
                                                                      __ushort_as_half(static_cast<unsigned short>(raw))))
                                                                : raw << 16;
            if (e < kEntries)
                reinterpret_cast<uint2*>(extra)[e % C::kStretches * (16 * MT + 8) + e / C::kStretches] =
                    make_uint2(sc, 0x43004300u | z | (z << 16));
        }
        if (r + kFewWarps < runs) load_group(r + kFewWarps);
        const int ahead = r + (C::kDepth - 1) * kFewWarps;
        if (lane == 0 && ahead < runs) issue(ahead, slot == 0 ? C::kDepth - 1 : slot - 1);
        if (!mbar_wait(bar0 + 8 * slot, phase, p.timeout_ns)) failed = true;
        if (__any_sync(0xffffffffu, failed)) {
            failed = true;
            break;
        }
        const uint8_t* unit = ring + slot * C::kUnit;
        if constexpr (PACK) {
            // Each lane cuts eight of a row's values, once for the run: piece lane / 4, word t = lane % 4.
#pragma unroll
            for (int m = 0; m < PACK; ++m) {
                const float4* x = reinterpret_cast<const float4*>(unit + C::kWeightBytes + m * kRun * 4) + 2 * lane;
                const float4 lo = x[0], hi = x[1];
                float u[4] = {lo.x, lo.y, lo.z, lo.w}, v[4] = {hi.x, hi.y, hi.z, hi.w};
                uint4* parts = reinterpret_cast<uint4*>(extra + C::kScaleBytes) + (g * 3 * PACK + 3 * m) * 4 + t;
#pragma unroll
                for (int q = 0; q < 3; ++q)
                    parts[q * 4] = make_uint4(cut_pair(u[0], v[0]), cut_pair(u[1], v[1]), cut_pair(u[2], v[2]),
                                              cut_pair(u[3], v[3]));
            }
            __syncwarp();
        }
        float acc[MT][RT][4] = {};
#pragma unroll
        for (int c = 0; c < kPieces; ++c) {
            // Parts of this lane's eight activations: pairs (k, k + 4) as the nibbles of a word pair up.
            uint32_t b[RT][PACK ? 1 : 3][4];
            if (PACK) {
                const uint4 v = reinterpret_cast<const uint4*>(extra + C::kScaleBytes)[part_at + c * 3 * PACK * 4];
                b[0][0][0] = v.x;
                b[0][0][1] = v.y;
                b[0][0][2] = v.z;
                b[0][0][3] = v.w;
            } else {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    const uint8_t* x = unit + C::kWeightBytes + c * C::kPieceBytes + (rt * 8 + g) * 128;
                    const float4 lo = *reinterpret_cast<const float4*>(x + (((2 * t) ^ g) << 4));
                    const float4 hi = *reinterpret_cast<const float4*>(x + (((2 * t + 1) ^ g) << 4));
                    float u[4] = {lo.x, lo.y, lo.z, lo.w}, v[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                    for (int q = 2; q >= 0; --q)  // (small parts first below)
#pragma unroll
                        for (int i = 0; i < 4; ++i) b[rt][PACK ? 0 : q][i] = cut_pair(u[i], v[i]);
                }
            }
            const int stretch = c >> SHIFT;
            const bool flush = ((c + 1) >> SHIFT) != stretch;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                uint32_t w[2];
                uint2 sz[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    w[h] = *reinterpret_cast<const uint32_t*>(unit + w_at[c] + (mt * 16 + h * 8) * (kRun / 2));
                    sz[h] = scale_at[stretch * (16 * MT + 8) + mt * 16 + h * 8];
                }
                const uint32_t a1[4] = {weight_pair(w[0], sz[0].y), weight_pair(w[1], sz[1].y),
                                        weight_pair(w[0] >> 4, sz[0].y), weight_pair(w[1] >> 4, sz[1].y)};
                const uint32_t a2[4] = {weight_pair(w[0] >> 8, sz[0].y), weight_pair(w[1] >> 8, sz[1].y),
                                        weight_pair(w[0] >> 12, sz[0].y), weight_pair(w[1] >> 12, sz[1].y)};
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
                    for (int q = 0; q < (PACK ? 1 : 3); ++q) {
                        mma_bf16(acc[mt][rt], a1, b[rt][q][0], b[rt][q][1]);
                        mma_bf16(acc[mt][rt], a2, b[rt][q][2], b[rt][q][3]);
                    }
                    if (flush) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            tot[mt][rt][i] += __uint_as_float(sz[i >> 1].x) * acc[mt][rt][i];
                            acc[mt][rt][i] = 0.0f;
                        }
                    }
                }
            }
        }
        if (++slot == C::kDepth) { slot = 0; phase ^= 1u; }
    }
    if (failed && lane == 0) {
        // Record it, and wait (again with a limit) for the copies still on their way to this CTA.
        atomicOr(p.err, kErrProducer);
        *abort_flag = 1;
        for (int d = 0; d < C::kDepth; ++d) {
            mbar_wait(bar0 + 8 * d, 0, p.timeout_ns);
            mbar_wait(bar0 + 8 * d, 1, p.timeout_ns);
        }
    }
    __syncthreads();  // every warp is done with the ring
    if (*abort_flag) return;
    // The warps' sums: [warp][MMA column][weight column], added in warp order (PACK: small parts first).
    float* red = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                red[(warp * 8 * RT + rt * 8 + 2 * t + (i & 1)) * 16 * MT + mt * 16 + (i >> 1) * 8 + g] = tot[mt][rt][i];
    __syncthreads();
    for (int i = threadIdx.x; i < rows * 16 * MT; i += 32 * kFewWarps) {
        const int m = i / (16 * MT), n = i % (16 * MT);
        if (n0 + n >= p.N) continue;
        float v = 0.0f;
#pragma unroll
        for (int q = PACK ? 2 : 0; q >= 0; --q)
#pragma unroll
            for (int w = 0; w < kFewWarps; ++w)
                v += red[(w * 8 * RT + (PACK ? 3 * m + q : m)) * 16 * MT + n];
        p.out[(m0 + m) * p.ldo + n0 + n] = apply_cell(v, m0 + m, n0 + n, 0, p.epi);
    }
}

template <int PACK, int RT, int MT, int SHIFT>
cudaError_t run_few_rows(const Q4Params& p, cudaStream_t stream) {
    using C = FewCfg<PACK, RT, MT, SHIFT>;
    auto kernel = q4_few_rows_kernel<PACK, RT, MT, SHIFT>;
    static std::mutex mu;
    static uint64_t configured = 0;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    {
        std::lock_guard<std::mutex> lock(mu);
        if (dev >= 64 || !(configured & (1ull << dev))) {
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
            if (e != cudaSuccess) return e;
            if (dev < 64) configured |= 1ull << dev;
        }
    }
    CUtensorMap mw, ma;
    const unsigned long long w_dims[2] = {static_cast<unsigned long long>(p.ldq), static_cast<unsigned long long>(p.N)};
    const unsigned long long w_stride[1] = {static_cast<unsigned long long>(p.ldq)};
    const unsigned w_box[2] = {C::kRun / 2, 16 * MT};
    const unsigned long long a_dims[2] = {static_cast<unsigned long long>(p.K), static_cast<unsigned long long>(p.M)};
    const unsigned long long a_stride[1] = {static_cast<unsigned long long>(p.lda) * 4};
    const unsigned a_box[2] = {PACK ? C::kRun : 32, C::kRows};
    if (!encode_tensor_map(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, p.q, w_dims, w_stride, w_box,
                           C::kRun == 256 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_128B) ||
        !encode_tensor_map(&ma, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, p.a, a_dims, a_stride, a_box,
                           PACK ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_128B))
        return cudaErrorInvalidValue;
    kernel<<<dim3((p.N + 16 * MT - 1) / (16 * MT), (p.M + C::kRows - 1) / C::kRows), 32 * kFewWarps, C::kSmem, stream>>>(
        mw, ma, p);
    note_launch();
    return cudaGetLastError();
}

template <int PACK, int RT, int MT>
cudaError_t run_few_rows_groups(const Q4Params& p, cudaStream_t stream) {
    // A scaling for every 128 k where the groups allow it, else for every 32.
    return p.group % 128 == 0 ? run_few_rows<PACK, RT, MT, 2>(p, stream) : run_few_rows<PACK, RT, MT, 0>(p, stream);
}

template <int PACK, int RT>
cudaError_t run_few_rows_width(const Q4Params& p, int num_sms, cudaStream_t stream) {
    // Wider warp tiles cut each activation for more weights; narrow ones fill the SMs.
    static const char* force = getenv("Q4_MT");
    if (force) {
        if (force[0] == '4') return run_few_rows_groups<PACK, RT, 4>(p, stream);
        if (force[0] == '2') return run_few_rows_groups<PACK, RT, 2>(p, stream);
        return run_few_rows_groups<PACK, RT, 1>(p, stream);
    }
    if (p.N >= 64 * num_sms && !PACK) return run_few_rows_groups<PACK, RT, 4>(p, stream);
    return p.N >= 32 * num_sms ? run_few_rows_groups<PACK, RT, 2>(p, stream) : run_few_rows_groups<PACK, RT, 1>(p, stream);
}

int q4_gemm(GpuCtx* ctx, Q4Params& p, const mxb_ep_step* steps, int n_steps, void* stream) {
    if (!ctx || !p.a || !p.q || !p.scales || !p.out || p.M < 1 || p.N < 1 || p.K < 1 || p.lda < p.K || p.ldo < p.N ||
        p.group < 32 || p.group % 32 || n_steps < 0 || n_steps > MXB_MAX_EPILOGUE || (n_steps > 0 && !steps) ||
        p.scale_type < MXB_SCALE_F32 || p.scale_type > MXB_SCALE_BF16) {
        set_error("mxb_q4_gemm: invalid arguments");
        return MXB_E_ARG;
    }
    if (p.ldq < (static_cast<long long>(p.K) + 1) / 2 || p.lds < (static_cast<long long>(p.K) + p.group - 1) / p.group) {
        set_error("mxb_q4_gemm: a weight row needs (K + 1) / 2 bytes and ceil(K / group) scales");
        return MXB_E_ARG;
    }
    const uintptr_t scale_mask = p.scale_type == MXB_SCALE_F32 ? 3 : 1;
    if (p.lda % 4 || (reinterpret_cast<uintptr_t>(p.a) & 15) || p.ldq % 16 || (reinterpret_cast<uintptr_t>(p.q) & 15) ||
        (reinterpret_cast<uintptr_t>(p.scales) & scale_mask)) {
        set_error("mxb_q4_gemm: A and Q need 16-byte aligned bases and row pitches (lda %% 4 == 0, ldq %% 16 == 0)");
        return MXB_E_ARG;
    }
    if (!take_cell_steps("mxb_q4_gemm", steps, n_steps, p.N, false, p.epi)) return MXB_E_ARG;
    DeviceScope scope(ctx->device);
    cudaStream_t st = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
    p.timeout_ns = ctx->timeout_ns;
    p.err = ctx->d_err;
    const cudaError_t e = p.M == 1   ? run_few_rows_width<1, 1>(p, ctx->num_sms, st)
                          : p.M == 2 ? run_few_rows_width<2, 1>(p, ctx->num_sms, st)
                          : p.M <= 8 ? run_few_rows_width<0, 1>(p, ctx->num_sms, st)
                                     : run_few_rows_width<0, 2>(p, ctx->num_sms, st);
    return cuda_ok(e, "4-bit product launch") ? MXB_OK : MXB_E_CUDA;
}

}  // namespace
}  // namespace mxb

extern "C" int mxb_q4_gemm(GpuCtx* ctx, const float* A, long long lda, const unsigned char* Q, long long ldq,
                           const void* scales, int scale_type, const unsigned char* zeros, long long lds, int group,
                           float* out, long long ldo, int M, int N, int K, const mxb_ep_step* steps, int n_steps,
                           void* stream) {
    try {
        mxb::Q4Params p{A, lda, Q, ldq, scales, zeros, lds, scale_type, group, out, ldo, M, N, K, 0, nullptr, {}};
        return mxb::q4_gemm(ctx, p, steps, n_steps, stream);
    } catch (const std::exception& e) {  // host allocations of the pool's lists
        mxb::set_error("mxb_q4_gemm: %s", e.what());
        return MXB_E_NOMEM;
    }
}
