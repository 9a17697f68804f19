// Products with 4-bit weights and group scales (mxb_q4_gemm):
//   out[m, n] = epi(sum over groups g of s[n, g] * sum over k in g of A[m, k] * (q[n, k] - z[n, g])).
#include "gemm_common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <exception>
#include <type_traits>

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
//
// Calls one behind the other, weights past L2: 1 x 4096 x 4096 5.6 us, 1 x 8192 x
// 8192 13.7 us (2.6 TB/s), 8 x 8192 x 8192 with groups of 32, fp32 scales and zero
// points 26.3 us (1.7 TB/s).  What bounds it there are the
// instructions that make bf16 pairs of nibbles and scale each group's sums:
// 54% of the issue slots and 48% of the ALU's.

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

// The top eight bits of x and y as a bf16 pair; x and y keep the rest.  Of an infinite value the rest would be inf - inf;
// INF: it keeps nothing instead (that is asked of the first part only, since what it leaves is finite or NaN).
template <bool INF>
__device__ __forceinline__ uint32_t cut_pair(float& x, float& y) {
    const uint32_t ux = __float_as_uint(x), uy = __float_as_uint(y);
    const float tx = __uint_as_float(ux & 0xFFFF0000u), ty = __uint_as_float(uy & 0xFFFF0000u);
    x = INF && x == tx ? 0.0f : x - tx;
    y = INF && y == ty ? 0.0f : y - ty;
    return __byte_perm(ux, uy, 0x7632);
}

// The next part of the pairs (u[i], v[i]).
template <bool INF>
__device__ __forceinline__ uint4 cut_pairs(float (&u)[4], float (&v)[4]) {
    return make_uint4(cut_pair<INF>(u[0], v[0]), cut_pair<INF>(u[1], v[1]), cut_pair<INF>(u[2], v[2]), cut_pair<INF>(u[3], v[3]));
}

// A scale as it lies in memory, and as a number: apart, so that a load can be under way while others are used.
__device__ __forceinline__ uint32_t scale_raw(const Q4Params& p, long long at) {
    return p.scale_type == MXB_SCALE_F32 ? ld_global(static_cast<const uint32_t*>(p.scales) + at)
                                         : ld_global(static_cast<const unsigned short*>(p.scales) + at);
}
__device__ __forceinline__ float scale_value(const Q4Params& p, uint32_t raw) {
    return p.scale_type == MXB_SCALE_F32   ? __uint_as_float(raw)
           : p.scale_type == MXB_SCALE_F16 ? __half2float(__ushort_as_half(static_cast<unsigned short>(raw)))
                                           : __uint_as_float(raw << 16);
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
    wait_for_previous_kernel();
    let_next_kernel_in();

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
                s_raw[i] = scale_raw(p, at);
                if (p.zeros) z_raw[i] = ld_global(p.zeros + at);
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
    int slot = 0;
    uint32_t phase = 0;
    bool failed = false;
    // This warp's sums of its runs; INF: with parts made so that an infinity stays one.
    auto sum_runs = [&](auto inf, float (&tot)[MT][RT][4]) {
        constexpr bool INF = decltype(inf)::value;
        int r = warp;
        if (lane == 0) {
#pragma unroll
            for (int d = 0; d < C::kDepth - 1; ++d)
                if (r + d * kFewWarps < runs) issue(r + d * kFewWarps, INF ? (slot + d) % C::kDepth : d);
        }
        if (r < runs) load_group(r);
        for (; r < runs; r += kFewWarps) {
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
                    for (int q = 0; q < 3; ++q) parts[q * 4] = cut_pairs<INF>(u, v);
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
                            for (int i = 0; i < 4; ++i) b[rt][PACK ? 0 : q][i] = cut_pair<INF>(u[i], v[i]);
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
    };
    // The warps' sums added in warp order (PACK: small parts first), each for `store`: its thread's j-th, row m and column n.
    float* red = reinterpret_cast<float*>(smem);  // [warp][MMA column][weight column]
    auto finish = [&](const float (&tot)[MT][RT][4], auto store) {
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
            store(i / (32 * kFewWarps), m, n, v);
        }
    };
    auto put = [&](int m, int n, float v) { p.out[(m0 + m) * p.ldo + n0 + n] = apply_cell(v, m0 + m, n0 + n, 0, p.epi); };
    uint32_t again = 0;  // this thread's outputs that are NaN
    {
        float tot[MT][RT][4] = {};
        sum_runs(std::false_type{}, tot);
        finish(tot, [&](int j, int m, int n, float v) {
            if (v != v) {
                again |= 1u << j;
            } else {
                put(m, n, v);
            }
        });
    }
    // NaN may be the parts inf and inf - inf of an infinite activation: those sums are made once more, with cuts that ask for
    // infinities.  Asking in every call costs 8 x 8192 x 8192 with groups of 32 28.6 us instead of 26.5 by a choice for each
    // value, 27.7 by a branch for every eight (16 rows 35.2 and 39.6 instead of 34.2).
    if (__syncthreads_or(again != 0)) {
        fence_proxy_async_shared();  // the sums in the ring, before copies are written over them
        __syncthreads();
        float tot[MT][RT][4] = {};
        sum_runs(std::true_type{}, tot);
        finish(tot, [&](int j, int m, int n, float v) {
            if (again >> j & 1) put(m, n, v);
        });
    }
}

// What the copies read of a weight row: not its pitch, behind whose last row the caller's memory may end.
unsigned long long weight_row_bytes(const Q4Params& p) { return (static_cast<unsigned long long>(p.K) + 1) / 2; }

template <int PACK, int RT, int MT, int SHIFT>
cudaError_t run_few_rows(const Q4Params& p, cudaStream_t stream) {
    using C = FewCfg<PACK, RT, MT, SHIFT>;
    const cudaError_t e = allow_shared<q4_few_rows_kernel<PACK, RT, MT, SHIFT>>(C::kSmem);
    if (e != cudaSuccess) return e;
    CUtensorMap mw, ma;
    const unsigned long long w_dims[2] = {weight_row_bytes(p), static_cast<unsigned long long>(p.N)};
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
    return launch_early(q4_few_rows_kernel<PACK, RT, MT, SHIFT>,
                        dim3((p.N + 16 * MT - 1) / (16 * MT), (p.M + C::kRows - 1) / C::kRows), dim3(32 * kFewWarps), C::kSmem,
                        stream, 1, mw, ma, p);
}

template <int PACK, int RT, int MT>
cudaError_t run_few_rows_groups(const Q4Params& p, cudaStream_t stream) {
    // A scaling for every 128 k where the groups allow it, else for every 32.
    return p.group % 128 == 0 ? run_few_rows<PACK, RT, MT, 2>(p, stream) : run_few_rows<PACK, RT, MT, 0>(p, stream);
}

template <int PACK, int RT>
cudaError_t run_few_rows_width(const Q4Params& p, int num_sms, cudaStream_t stream) {
    // Wider warp tiles cut each activation for more weights; narrow ones fill the SMs.  8192 x 8192, groups
    // of 128, cold L2: one row 25.4 / 19.5 us at 16 / 32 columns a warp, eight rows 37.9 / 29.6 / 27.6 us at
    // 16 / 32 / 64 (groups of 32: 42.0 / 31.7 / 33.8), sixteen rows 68.6 / 46.0 / 35.8 us.
    if (RT == 2 && p.N >= 32 * num_sms) return run_few_rows_groups<PACK, RT, RT == 2 ? 4 : 2>(p, stream);
    return p.N >= 24 * num_sms ? run_few_rows_groups<PACK, RT, 2>(p, stream) : run_few_rows_groups<PACK, RT, 1>(p, stream);
}

// ---------------------------------------------------------------- many rows
//
// More than 16 rows: bound by the tensor cores.  A tile is 128 weight columns
// (TMEM lanes) by up to 128 rows (TMEM columns).  Eight warps, a thread to a
// weight column, turn the 4-bit values of 64 k into bf16 q - z (exact) in
// tensor memory, the MMA's A operand; the activations' three bf16 parts, cut
// beforehand into workspace by q4_cut_kernel, arrive by TMA; per 16 k the three
// parts are multiplied into the same accumulator.  That is 3 bf16 products,
// half the tensor time of the 3xTF32 product that fp32 weights need, and exact
// up to the fp32 sums.  With the weights in shared memory as well, its 128 bytes
// a clock were the limit (164 KB a stage against 768 clocks of MMA; now 104 KB).
// An accumulator takes the k of one group (at most 128); the epilogue warps,
// whose lanes each hold one weight column, add it times that column's scale to
// fp32 totals.
// The eight k of a word keep the order in which its nibbles pair up (k, k + 4):
// the cut kernel writes the activations in the same order.
// With fewer tiles than SMs, a cluster of `splits` CTAs shares a tile, each
// summing its own stretch of K; the totals meet in distributed shared memory,
// added in CTA order.
//
// 1000 x 8192 x 8192, groups of 128: 324 us in a burst (414 TFLOP/s, 1243 of the
// tensor core's bf16 ones), 346-380 us once the power limit has the clock at 1.57
// GHz; the tensor cores are then 65% active.

constexpr int kManyCols = 128;  // rows of A per tile, at most
constexpr int kManyK = 64;      // k per stage: 128 bytes of bf16

struct ManyCfg {
    static constexpr int kXBytes = 3 * kManyCols * kManyK * 2;  // the parts of a stage
    static constexpr int kXStages = 4;
    static constexpr int kRawBytes = 128 * 64;                  // 128 k of 128 weight rows
    static constexpr int kRawStages = 3;
    static constexpr int kDeqStages = 4;                        // weights in tensor memory: 32 columns each
    static constexpr int kEpiWarps = 8, kConvWarps = 8;
    static constexpr int kThreads = 32 * (kEpiWarps + kConvWarps + 4);  // and a warpgroup with TMA and MMA
    // Registers a thread: the launch has 640 x 96, given out in shares of 128 threads.
    static constexpr int kEpiRegs = 160, kConvRegs = 56, kIssueRegs = 48;
    static_assert(2 * kEpiRegs + 2 * kConvRegs + kIssueRegs <= 480, "more registers than the launch has");
    static constexpr int kRawOffset = kXStages * kXBytes;
    static constexpr int kBarOffset = kRawOffset + kRawStages * kRawBytes;
    static constexpr int kNumBars = 2 * kXStages + 2 * kRawStages + 2 * kDeqStages + 4 + 1;
    static constexpr int kDeqCol = 2 * kManyCols;               // first TMEM column behind the two accumulators
    static constexpr int kTmemCols = 512;
    static constexpr int kSmem = 1024 + kBarOffset + kNumBars * 8 + 16;
    static constexpr int kMaxSplits = 8;
    static_assert(kDeqCol + 32 * kDeqStages <= kTmemCols, "tensor memory");
    static_assert(kManyCols * 128 * 4 <= kRawOffset, "a tile's totals fit in the activations' stages");
    static_assert(kSmem <= 227 * 1024, "shared memory budget");
};

// kind::f16 with bf16 operands, both K-major, fp32 accumulation.
__host__ __device__ constexpr uint32_t idesc_bf16(int m, int n) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) |
           (static_cast<uint32_t>(m >> 4) << 24);
}

// A in tensor memory: lane i holds row i, a 32-bit column two elements along K.  The whole warp comes here and one
// thread issues (`leader`): without a branch around it the operands stay in uniform registers, which the instruction
// reads, instead of being moved there for every MMA.
__device__ __forceinline__ void mma_f16_ts(uint32_t leader, uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc,
                                           uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(leader)
        : "memory");
}

// parts[q][m][k'] = part q of A[m][k], k' the pair order within each eight k; zeros from K to kp.
__global__ void __launch_bounds__(256) q4_cut_kernel(const float* a, long long lda, int M, int K, long long kp,
                                                     uint4* parts) {
    const long long eights = kp / 8, total = M * eights;
    wait_for_previous_kernel();
    let_next_kernel_in();
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
        const long long m = i / eights;
        const int k = static_cast<int>(i - m * eights) * 8;
        const float* src = a + m * lda + k;
        float u[4], v[4];
        if (k + 8 <= K) {
            const float4 lo = ld_global(reinterpret_cast<const float4*>(src));
            const float4 hi = ld_global(reinterpret_cast<const float4*>(src) + 1);
            u[0] = lo.x, u[1] = lo.y, u[2] = lo.z, u[3] = lo.w;
            v[0] = hi.x, v[1] = hi.y, v[2] = hi.z, v[3] = hi.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                u[j] = k + j < K ? ld_global(src + j) : 0.0f;
                v[j] = k + 4 + j < K ? ld_global(src + 4 + j) : 0.0f;
            }
        }
        parts[i] = cut_pairs<true>(u, v);
        parts[total + i] = cut_pairs<false>(u, v);
        parts[2 * total + i] = cut_pairs<false>(u, v);
    }
}

struct ManyParams {
    Q4Params q;
    int cols;              // rows of A per tile: a multiple of 16
    int col_tiles, tiles;
    int splits;
};

__device__ __forceinline__ void raise_q4(const Q4Params& p, volatile int* abort_flag, int bit) {
    atomicOr(p.err, bit);
    *abort_flag = 1;
}

// The group of successive k, without a division for each.
struct GroupWalk {
    int group, index, pos;  // pos: k - index * group
    __device__ __forceinline__ void step(int k) {
        for (pos += k; pos >= group; pos -= group) ++index;
    }
};

__global__ void __launch_bounds__(ManyCfg::kThreads, 1)
    q4_many_rows_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
                        const __grid_constant__ ManyParams mp) {
    using C = ManyCfg;
    const Q4Params& p = mp.q;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kBarOffset);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::kNumBars);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const uint32_t bar0 = smem_addr(bars);
    constexpr int kX = C::kXStages, kR = C::kRawStages, kD = C::kDeqStages;
    auto xfull = [&](int s) { return bar0 + 8u * s; };
    auto xempty = [&](int s) { return bar0 + 8u * (kX + s); };
    auto rfull = [&](int s) { return bar0 + 8u * (2 * kX + s); };
    auto rempty = [&](int s) { return bar0 + 8u * (2 * kX + kR + s); };
    auto dfull = [&](int s) { return bar0 + 8u * (2 * kX + 2 * kR + s); };
    auto dempty = [&](int s) { return bar0 + 8u * (2 * kX + 2 * kR + kD + s); };
    auto tfull = [&](int a) { return bar0 + 8u * (2 * kX + 2 * kR + 2 * kD + a); };
    auto tempty = [&](int a) { return bar0 + 8u * (2 * kX + 2 * kR + 2 * kD + 2 + a); };
    const uint32_t drain = bar0 + 8u * (2 * kX + 2 * kR + 2 * kD + 4);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int kConvWarp = C::kEpiWarps, kTmaWarp = kConvWarp + C::kConvWarps, kMmaWarp = kTmaWarp + 1;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kX; ++s) {
            mbar_init(xfull(s), 1);
            mbar_init(xempty(s), 1);
        }
        for (int s = 0; s < kR; ++s) {
            mbar_init(rfull(s), 1);
            mbar_init(rempty(s), C::kConvWarps);
        }
        for (int s = 0; s < kD; ++s) {
            mbar_init(dfull(s), C::kConvWarps);
            mbar_init(dempty(s), 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(tfull(a), 1);
            mbar_init(tempty(a), C::kEpiWarps);
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_barrier_init();
        tma_prefetch_desc(&tm_w);
        tma_prefetch_desc(&tm_x);
    }
    if (warp == kMmaWarp) {
        tmem_alloc(smem_addr(tmem_slot), C::kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    wait_for_previous_kernel();
    let_next_kernel_in();

    const int all_stages = (p.K + kManyK - 1) / kManyK;
    const int halves = (p.K + 31) / 32;                                     // of 32 k
    const int seg = p.group % 128 == 0 ? 4 : p.group % 64 == 0 ? 2 : 1;     // halves to an accumulator
    const int team = blockIdx.x / mp.splits, teams = gridDim.x / mp.splits, rank = blockIdx.x - team * mp.splits;
    // This CTA's stages [kb0, kb1) of every tile: whole runs of 128 k, so that no accumulator crosses a group.
    const int runs = (all_stages + 1) / 2;
    const int kb0 = static_cast<int>(static_cast<long long>(runs) * rank / mp.splits) * 2;
    const int kb1 = min(all_stages, static_cast<int>(static_cast<long long>(runs) * (rank + 1) / mp.splits) * 2);

    if (warp >= kTmaWarp) {
      fewer_registers<C::kIssueRegs>();
      if (warp == kTmaWarp) {
        // ------------------------------------------------------------ TMA producer
        const bool leader = elect_one();
        const uint32_t x_bytes = static_cast<uint32_t>(3 * mp.cols * kManyK * 2);
        int xs = 0, rs = 0;
        uint32_t xph = 0, rph = 0;
        long long xn = 0, rn = 0;
        bool ok = true;
        for (int t = team; t < mp.tiles && ok; t += teams) {
            const int n0 = t / mp.col_tiles * 128, m0 = t % mp.col_tiles * mp.cols;
            for (int kb = kb0; kb < kb1; ++kb) {
                if ((kb & 1) == 0) {
                    if (*abort_flag || !mbar_wait(rempty(rs), rph ^ 1u, p.timeout_ns)) {
                        ok = false;
                        break;
                    }
                    if (leader) {
                        mbar_arrive_expect_tx(rfull(rs), C::kRawBytes);
                        tma_load_2d(smem_addr(smem + C::kRawOffset + rs * C::kRawBytes), &tm_w, rfull(rs), kb * 32, n0);
                    }
                    __syncwarp();
                    ++rn;
                    if (++rs == kR) { rs = 0; rph ^= 1u; }
                }
                if (*abort_flag || !mbar_wait(xempty(xs), xph ^ 1u, p.timeout_ns)) {
                    ok = false;
                    break;
                }
                if (leader) {
                    mbar_arrive_expect_tx(xfull(xs), x_bytes);
                    tma_load_3d(smem_addr(smem + xs * C::kXBytes), &tm_x, xfull(xs), kb * kManyK, m0, 0);
                }
                __syncwarp();
                ++xn;
                if (++xs == kX) { xs = 0; xph ^= 1u; }
            }
        }
        if (!ok && leader) {
            raise_q4(p, abort_flag, kErrProducer);
            // Copies in flight land in this CTA's shared memory: wait for them before leaving.
            for (long long i = xn > kX ? xn - kX : 0; i < xn; ++i)
                mbar_wait(xfull(static_cast<int>(i % kX)), static_cast<uint32_t>((i / kX) & 1), p.timeout_ns);
            for (long long i = rn > kR ? rn - kR : 0; i < rn; ++i)
                mbar_wait(rfull(static_cast<int>(i % kR)), static_cast<uint32_t>((i / kR) & 1), p.timeout_ns);
        }
        __syncwarp();
      } else if (warp == kMmaWarp) {
        // ------------------------------------------------------------ MMA issuer
        constexpr uint32_t kHi = smem_desc_hi(1024, kLayoutSW128);
        const bool leader = elect_one();
        int xs = 0, ds = 0, acc = 0;
        uint32_t xph = 0, dph = 0, aph = 0;
        bool ok = true;
        for (int t = team; t < mp.tiles && ok; t += teams) {
            const int m0 = t % mp.col_tiles * mp.cols;
            const uint32_t idesc = idesc_bf16(128, (min(mp.cols, p.M - m0) + 15) & ~15);
            const uint32_t part = static_cast<uint32_t>(mp.cols * 8);  // 128 bytes a row, in descriptor steps of 16
            int in_seg = 0;
            for (int kb = kb0; kb < kb1 && ok; ++kb) {
                if (*abort_flag || !mbar_wait(xfull(xs), xph, p.timeout_ns) ||
                    !mbar_wait(dfull(ds), dph, p.timeout_ns)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t w = tmem_base + static_cast<uint32_t>(C::kDeqCol + 32 * ds);
                const uint32_t x = smem_desc_lo(smem_addr(smem + xs * C::kXBytes), 16);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (2 * kb + h >= halves) break;
                    if (in_seg == 0) {
                        if (!mbar_wait(tempty(acc), aph ^ 1u, p.timeout_ns)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                    }
                    const uint32_t d = tmem_base + static_cast<uint32_t>(acc * kManyCols);
#pragma unroll
                    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                        for (int q = 2; q >= 0; --q)  // small parts first
                            mma_f16_ts(leader, d, w + 8 * (2 * h + kk), smem_desc_of(kHi, x + q * part + 2 * (2 * h + kk)),
                                       idesc, kk == 0 && q == 2 ? (in_seg != 0 ? 1u : 0u) : 1u);
                    if (++in_seg == seg || 2 * kb + h == min(2 * kb1, halves) - 1) {
                        if (leader) mma_commit(tfull(acc));
                        in_seg = 0;
                        acc ^= 1;
                        if (acc == 0) aph ^= 1u;
                    }
                }
                if (leader) {
                    mma_commit(xempty(xs));
                    mma_commit(dempty(ds));
                }
                if (++xs == kX) { xs = 0; xph ^= 1u; }
                if (++ds == kD) { ds = 0; dph ^= 1u; }
            }
        }
        if (leader) {
            if (!ok) raise_q4(p, abort_flag, kErrMma);
            mma_commit(drain);
            if (!mbar_wait(drain, 0, p.timeout_ns)) raise_q4(p, abort_flag, kErrMma);
        }
        __syncwarp();
      }
    } else if (warp >= kConvWarp) {
        // ------------------------------------------------------------ 4 bits to bf16: a weight column and 32 k a thread
        fewer_registers<C::kConvRegs>();
        const int tid = threadIdx.x - 32 * kConvWarp, row = tid & 127, half = tid >> 7;
        const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(row & ~31) << 16) + C::kDeqCol + 16 * half;
        int rs = 0, ds = 0;
        uint32_t rph = 0, dph = 0;
        bool failed = false;
        for (int t = team; t < mp.tiles && !failed; t += teams) {
            const int n = min(t / mp.col_tiles * 128 + row, p.N - 1);
            GroupWalk at{p.group, 0, 0};
            at.step(kb0 * kManyK + 32 * half);
            auto zero_of = [&](int kb) -> uint32_t {
                return p.zeros && kb * kManyK + 32 * half < p.K ? ld_global(p.zeros + n * p.lds + at.index) : 8u;
            };
            uint32_t z_next = zero_of(kb0);
            for (int kb = kb0; kb < kb1; ++kb) {
                const uint32_t z = z_next & 15u;
                at.step(kManyK);
                if (kb + 1 < kb1) z_next = zero_of(kb + 1);
                const bool stop = __any_sync(0xffffffffu, *abort_flag != 0);
                const bool got = !stop && mbar_wait(rfull(rs), rph, p.timeout_ns) &&
                                 mbar_wait(dempty(ds), dph ^ 1u, p.timeout_ns);
                if (!__all_sync(0xffffffffu, got)) {
                    if (lane == 0 && !stop) raise_q4(p, abort_flag, kErrProducer);
                    failed = true;
                    break;
                }
                const int chunk = (kb & 1) * 2 + half;  // 16 bytes of the row's 64
                const uint4 w4 = *reinterpret_cast<const uint4*>(smem + C::kRawOffset + rs * C::kRawBytes + row * 64 +
                                                                 ((chunk ^ ((row >> 1) & 3)) << 4));
                const uint32_t z128 = 0x43004300u | z | (z << 16);
                const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
                uint32_t r[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) r[j] = weight_pair(w[j >> 2] >> (4 * (j & 3)), z128);
                tc_fence_after();
                tmem_st_32x32b_x16(lane_base + static_cast<uint32_t>(32 * ds), r);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(dfull(ds));
                    if ((kb & 1) || kb == kb1 - 1) mbar_arrive(rempty(rs));
                }
                if (++ds == kD) { ds = 0; dph ^= 1u; }
                if ((kb & 1) || kb == kb1 - 1) {
                    if (++rs == kR) { rs = 0; rph ^= 1u; }
                }
            }
        }
    } else {
        // ------------------------------------------------------------ epilogue: a weight column and 64 rows a thread
        // (Sixteen warps, with 32 rows a thread, were no faster: 606 against 620 us with groups of 32, 340 against 326 with
        // groups of 128.)
        more_registers<C::kEpiRegs>();
        constexpr int W = 16, kTotals = kManyCols / 2;
        const int quad = warp & 3, first_col = (warp >> 2) * kTotals;
        const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + first_col;
        int acc = 0;
        uint32_t aph = 0;
        bool failed = false;
        for (int t = team; t < mp.tiles && !failed; t += teams) {
            const int col = t / mp.col_tiles * 128 + quad * 32 + lane, m0 = t % mp.col_tiles * mp.cols;
            const int cols = min(mp.cols, p.M - m0);
            const long long scale_row = min(col, p.N - 1) * p.lds;
            float total[kTotals];
#pragma unroll
            for (int i = 0; i < kTotals; ++i) total[i] = 0.0f;
            GroupWalk at{p.group, 0, 0};
            at.step(kb0 * kManyK);
            uint32_t s_next = scale_raw(p, scale_row + at.index);
            const int h1 = min(2 * kb1, halves);
            for (int h = 2 * kb0; h < h1; h += seg) {
                const float s = scale_value(p, s_next);
                at.step(32 * seg);
                if (h + seg < h1) s_next = scale_raw(p, scale_row + at.index);
                const bool stop = __any_sync(0xffffffffu, *abort_flag != 0);
                const bool got = !stop && mbar_wait(tfull(acc), aph, p.timeout_ns);
                if (!__all_sync(0xffffffffu, got)) {
                    if (lane == 0 && !stop) raise_q4(p, abort_flag, kErrEpilogue);
                    failed = true;
                    break;
                }
                tc_fence_after();
                // The second half's load is under way while the first is added.
                const uint32_t src = lane_base + static_cast<uint32_t>(acc * kManyCols);
                if (first_col < cols) {
                    uint32_t r[32], q[32];
                    tmem_ld_32x32b_x32(src, r);
                    tmem_ld_wait();
                    if (first_col + 32 < cols) tmem_ld_32x32b_x32(src + 32, q);
#pragma unroll
                    for (int i = 0; i < 32; ++i) total[i] += s * __uint_as_float(r[i]);
                    if (first_col + 32 < cols) {
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 32; ++i) total[32 + i] += s * __uint_as_float(q[i]);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(tempty(acc));
                acc ^= 1;
                if (acc == 0) aph ^= 1u;
            }
            if (failed) break;
            if (mp.splits > 1) {
                // The one tile of this cluster: every copy and MMA of it is done, so the activations' stages can hold
                // the totals, [row][weight column].
                float* share = reinterpret_cast<float*>(smem) + first_col * 128 + quad * 32 + lane;
#pragma unroll
                for (int i = 0; i < kTotals; ++i) share[i * 128] = total[i];
                continue;
            }
            if (col < p.N) {
#pragma unroll
                for (int c = 0; c < kTotals; c += W) {
                    const int n = min(W, cols - first_col - c);
                    if (n <= 0) continue;
                    float v[W];
#pragma unroll
                    for (int i = 0; i < W; ++i) v[i] = total[c + i];
                    const long long row = m0 + first_col + c;
                    apply_column<W>(v, row, n, col, 0, p.epi);
                    float* dst = p.out + row * p.ldo + col;
#pragma unroll
                    for (int i = 0; i < W; ++i)
                        if (i < n) __stcs(dst + i * p.ldo, v[i]);
                }
            }
        }
    }

    if (mp.splits > 1) {
        __syncwarp();
        cluster_sync();  // the totals of every CTA of the tile are in place (or a CTA gave up)
        if (team < mp.tiles && *abort_flag == 0) {
            const int n0 = team / mp.col_tiles * 128, m0 = team % mp.col_tiles * mp.cols;
            // Every thread an output, this CTA the rows rank, rank + splits, ...
            const int share = (min(mp.cols, p.M - m0) - rank + mp.splits - 1) / mp.splits;
            for (int i = threadIdx.x; i < share * 128; i += C::kThreads) {
                const int row = rank + (i >> 7) * mp.splits, col = n0 + (i & 127);
                if (col >= p.N) continue;
                const uint32_t at = smem_addr(smem) + static_cast<uint32_t>(row * 128 + (i & 127)) * 4;
                float v = 0.0f;
                for (int r = 0; r < mp.splits; ++r) v += ld_shared_cluster_f32(mapa_shared(at, static_cast<uint32_t>(r)));
                p.out[(m0 + row) * p.ldo + col] = apply_cell(v, m0 + row, col, 0, p.epi);
            }
        }
        __syncwarp();
        cluster_sync();  // no CTA leaves while another still reads its totals
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem_base, C::kTmemCols);
    }
}

int run_many_rows(GpuCtx* ctx, const Q4Params& p, cudaStream_t stream) {
    using C = ManyCfg;
    if (!cuda_ok(allow_shared<q4_many_rows_kernel>(C::kSmem), "4-bit product set-up")) return MXB_E_CUDA;
    const long long kp = (static_cast<long long>(p.K) + kManyK - 1) / kManyK * kManyK;
    Scratch scratch(ctx, stream);
    void* parts = scratch.alloc(static_cast<size_t>(3) * p.M * kp * 2);
    if (!parts) return MXB_E_NOMEM;
    const long long blocks = (p.M * (kp / 8) + 255) / 256;
    if (!cuda_ok(launch_early(q4_cut_kernel, dim3(static_cast<unsigned>(std::min<long long>(blocks, 8ll * ctx->num_sms))),
                              dim3(256), 0, stream, 1, p.a, p.lda, p.M, p.K, kp, static_cast<uint4*>(parts)),
                 "4-bit product: cutting the rows"))
        return MXB_E_CUDA;

    // The tile width (a multiple of 16) that needs the least time in whole rounds of the SMs: a round costs its width (96
    // columns at least: a narrower MMA takes no less) and about 32 columns more.  1000 rows x 8192: 9 tiles of 112 in 4
    // rounds instead of 8 of 128 in 4.
    const long long lane_tiles = (p.N + 127) / 128;
    ManyParams mp{p, kManyCols, 0, 0, 1};
    long long best = -1;
    for (int w = kManyCols; w >= 16; w -= 16) {
        const long long rounds = ((p.M + w - 1) / w * lane_tiles + ctx->num_sms - 1) / ctx->num_sms;
        const long long cost = rounds * (std::max(w, 96) + 32);
        if (best < 0 || cost < best) {
            best = cost;
            mp.cols = w;
        }
    }
    mp.col_tiles = (p.M + mp.cols - 1) / mp.cols;
    const long long tiles = mp.col_tiles * lane_tiles;
    if (tiles >= (1ll << 31)) {
        set_error("mxb_q4_gemm: too many tiles");
        return MXB_E_UNSUPPORTED;
    }
    mp.tiles = static_cast<int>(tiles);
    // Splits while every cluster still has SMs of its own and every CTA at least two runs of 128 k.
    const int runs = (p.K + 127) / 128;
    while (mp.splits < C::kMaxSplits && 2 * mp.splits * tiles <= ctx->num_sms && runs >= 4 * mp.splits) mp.splits *= 2;
    CUtensorMap mw, mx;
    const unsigned long long w_dims[2] = {weight_row_bytes(p), static_cast<unsigned long long>(p.N)};
    const unsigned long long w_stride[1] = {static_cast<unsigned long long>(p.ldq)};
    const unsigned w_box[2] = {64, 128};
    const unsigned long long x_dims[3] = {static_cast<unsigned long long>(kp), static_cast<unsigned long long>(p.M), 3};
    const unsigned long long x_strides[2] = {static_cast<unsigned long long>(kp) * 2,
                                             static_cast<unsigned long long>(kp) * 2 * p.M};
    const unsigned x_box[3] = {kManyK, static_cast<unsigned>(mp.cols), 3};
    if (!encode_tensor_map(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, p.q, w_dims, w_stride, w_box,
                           CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B) ||
        !encode_tensor_map(&mx, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, parts, x_dims, x_strides, x_box,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B)) {
        set_error("mxb_q4_gemm: the tensor maps could not be made");
        return MXB_E_CUDA;
    }
    const dim3 grid(static_cast<unsigned>(mp.splits > 1 ? tiles * mp.splits : std::min<long long>(tiles, ctx->num_sms)));
    const cudaError_t e =
        launch_early(q4_many_rows_kernel, grid, dim3(C::kThreads), C::kSmem, stream, mp.splits, mw, mx, mp);
    return cuda_ok(e, "4-bit product launch") ? MXB_OK : MXB_E_CUDA;
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
    if (p.M > kMaxExtent || p.N > kMaxExtent || p.K > kMaxExtent) {
        set_error("mxb_q4_gemm: M, N and K are limited to 2^30");
        return MXB_E_UNSUPPORTED;
    }
    if (!take_cell_steps("mxb_q4_gemm", steps, n_steps, p.N, false, p.epi)) return MXB_E_ARG;
    DeviceScope scope(ctx->device);
    cudaStream_t st = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
    p.timeout_ns = ctx->timeout_ns;
    p.err = ctx->d_err;
    // 8192 x 8192, groups of 128, calls one behind the other: 16 rows 30 us in the few-row kernel, whose time grows with
    // every eight rows (8: 23); 17 rows 41 us in the other, whose time is nearly that of 96 (49).
    if (p.M > 16) return run_many_rows(ctx, p, st);
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
