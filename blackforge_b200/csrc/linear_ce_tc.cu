// The tcgen05 kernel behind the linear cross entropy (see linear_ce.cu for the operator): a CTA-pair GEMM
// (tcgen05.mma.cta_group::2, 256 x 256 output tiles, fp32 accumulators in tensor memory) whose epilogue never stores
// the logits.
//
//   kCeStats  z = x W^T + b per tile; each row's running maximum and sum of exponentials over the tile's columns
//             go to a small array (one pair per row and 128 columns), the label's logit to one word per row
//   kCeDz     the same product; the epilogue stores dz = w (exp(z - lse) - [column = label]) in bf16 for one piece of
//             the vocabulary, and column sums of the unrounded dz per 32 rows for the bias gradient. w is the row's own
//             weight only: a factor common to all rows (1 / rows) would give the label's entries, all near -1, one and
//             the same rounding error, which the sums over rows and columns cannot average away
//   kCeGrad   the products with dz times that common factor: dx += dz W (B operand with its reduction along rows) and dW = dz^T x (both
//             operands that way). The MN-major operand forms of tcgen05 read the tiles as they lie in memory, so
//             nothing is transposed by a pass of its own.
//
// Bound by the tensor pipe: of the measured cuBLAS rate the statistics reach 100 % (4096 x 32000 x 2048 in 0.323 ms), dz 98 %
// (16384 x 8192 x 2048 in 0.340 ms), dW 89 - 95 % and dx 95 % of it in isolation; a whole step of 16384 x 32000 x 2048 takes 5.5 ms
// (1555 TFLOP/s over its four products), 6.5 ms where steps follow each other and the power limit sets the clock. The tile is
// the 256 x 256 of a pair because its operands (64 B/clk read by the MMAs, 64 B/clk written by TMA) just fit the shared memory's
// bandwidth; an epilogue of two exponentials per logit and a row's 128 columns hides under a tile's MMAs from a depth of about 512.
//
// Roles, rings and barriers are those of the plain CTA-pair GEMM (gemm_tc2.cu): a TMA producer warp per CTA, one MMA
// issuer in the leader CTA, eight epilogue warps per CTA on double-buffered accumulators.
#include <cuda.h>
#include <cuda_bf16.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.hpp"
#include "linear_ce.cuh"
#include "ptx_sm100.cuh"

namespace bfb {

namespace {

constexpr int kCePairM = 256;                 // rows of a pair's tile, 128 per CTA
constexpr int kCeAccN = 256;                  // columns of a tile
constexpr int kCeBlockK = 64;                 // reduction depth per stage: one 128-byte swizzle row of bf16
constexpr int kCeRowBytes = 128;
constexpr int kCeOperandBytes = 128 * kCeRowBytes;      // 16 KiB: 128 rows (or columns) x 64 of A, the same of B
constexpr int kCeStageBytes = 2 * kCeOperandBytes;
constexpr int kCeStages = 6;
constexpr int kCeThreads = 384;               // producer, MMA, tensor-memory warp, spare + 8 epilogue warps
constexpr int kCeEpilogueWarps = 8;
constexpr int kCeSmemBytes = kCeStages * kCeStageBytes + 1024 + 256 + kCeEpilogueWarps * 4096;

enum { kCeStats = 0, kCeDz = 1, kCeGrad = 2 };

struct CeTile {
    int m, n;
};

__device__ __forceinline__ CeTile ceTileCoord(int t, int tilesM, int tilesN, int groupN) {
    const int fullGroups = tilesN / groupN;
    const int perGroup = tilesM * groupN;
    int g = t / perGroup;
    int width = groupN;
    int r = t - g * perGroup;
    if (g >= fullGroups) {
        g = fullGroups;
        r = t - fullGroups * perGroup;
        width = tilesN - fullGroups * groupN;
    }
    return {r / width, g * groupN + r % width};
}

struct CeEpilogue {
    // kCeStats, kCeDz
    const float* bias = nullptr;      // [vocab], at the piece's first column
    const float* labels = nullptr;    // [tokens]
    int64_t vocab = 0;                // whole vocabulary: labels at or above it do not count
    int64_t firstColumn = 0;          // vocabulary index of the piece's first column
    float2* partials = nullptr;       // [parts][tokens] (maximum, sum of exp(z - maximum)) per 128 columns
    float* labelLogit = nullptr;      // [tokens]
    const float* lse = nullptr;       // [tokens]
    const float* gradLoss = nullptr;  // [tokens] or null
    __nv_bfloat16* dz = nullptr;      // [tokens][ldDz]
    int64_t ldDz = 0;
    float* biasPartials = nullptr;    // [ceil(tokens / 32)][ldDz] or null
    // kCeGrad
    const float* dGradScale = nullptr;  // one word or null
    float gradScale = 1.0f;
    void* out = nullptr;              // [m][ldOut]
    int64_t ldOut = 0;
    const float* addend = nullptr;    // fp32 [m][ldAddend], or null: the sum over the pieces before this one
    int64_t ldAddend = 0;
};

// Sum over the warp's 32 lanes of 32 values per lane: lane j returns the sum of v[j]. Each exchange halves the values
// a lane still holds: 31 shuffles instead of 32 x 5.
__device__ __forceinline__ float warpColumnSums(float (&v)[32], int lane) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const bool upper = (lane & o) != 0;
#pragma unroll
        for (int j = 0; j < o; ++j) {
            const float keep = upper ? v[j + o] : v[j];
            const float give = upper ? v[j] : v[j + o];
            v[j] = keep + __shfl_xor_sync(0xFFFFFFFFu, give, o);
        }
    }
    return v[0];
}

// Columns [col, col + 32) of the accumulator as logits: bias added, columns at or behind `n` at -inf. Lane j fetches
// the word of column j once and hands it round.
__device__ __forceinline__ void ceLogits(const uint32_t (&raw)[32], float (&v)[32], const float* bias, int col, int n, int lane) {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(raw[j]);
    if (bias != nullptr || col + 32 > n) {
        const bool live = col + lane < n;
        const float b = !live ? -INFINITY : (bias != nullptr ? __ldg(bias + col + lane) : 0.0f);
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] += __shfl_sync(0xFFFFFFFFu, b, j);
    }
}

template <int kMode, bool kAMn, bool kBMn, typename TC>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kCeThreads, 1)
cePairKernel(const __grid_constant__ CUtensorMap tmapA, const __grid_constant__ CUtensorMap tmapB, const CeEpilogue ep, int m, int n,
             int k, int tilesM, int tilesN, int groupN, int kPerSplit, int splits, int* status) {
    constexpr uint32_t kIdesc = make_idesc(kCePairM, 256, 1u, kBMn ? 1u : 0u) | (kAMn ? 1u << 15 : 0u);

    extern __shared__ uint8_t smemRaw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smemRaw) + 1023) & ~uintptr_t(1023));
    uint64_t* fullBar = reinterpret_cast<uint64_t*>(smem + kCeStages * kCeStageBytes);
    uint64_t* emptyBar = fullBar + kCeStages;
    uint64_t* accFullBar = emptyBar + kCeStages;
    uint64_t* accEmptyBar = accFullBar + 2;
    uint32_t* tmemSlot = reinterpret_cast<uint32_t*>(accEmptyBar + 2);
    volatile int* abortFlag = reinterpret_cast<volatile int*>(tmemSlot + 1);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    const int numK = (k + kCeBlockK - 1) / kCeBlockK;
    const int tiles = tilesM * tilesN;
    const int totalTiles = tiles * splits;   // a tile's reduction in `splits` parts of kPerSplit stages
    const int clusterId = blockIdx.x >> 1;
    const int numClusters = gridDim.x >> 1;

    pdl_launch_dependents();   // the next kernel of the step may set itself up; it waits for this one's results
    if (threadIdx.x == 0) {
        for (int s = 0; s < kCeStages; ++s) {
            mbar_init(&fullBar[s], 1);
            mbar_init(&emptyBar[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&accFullBar[b], 1);
            mbar_init(&accEmptyBar[b], 2 * kCeEpilogueWarps);
        }
        *abortFlag = 0;
        fence_mbar_init();
        tma_prefetch_desc(&tmapA);
        tma_prefetch_desc(&tmapB);
    }
    if (warp == 2) {
        tmem_alloc(tmemSlot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();  // both CTAs' barriers exist before any remote arrival or copy can reach them
    tc_fence_after();
    const uint32_t tmemBase = *tmemSlot;
    pdl_wait();   // nothing of the kernel before is read, and nothing it reads overwritten, before here

    if (warp == 0) {
        // ---------------- TMA producer (both CTAs) ----------------
        int stage = 0;
        uint32_t phase = 0;
        bool alive = true;
        for (int t = clusterId; t < totalTiles && alive; t += numClusters) {
            const CeTile tc = ceTileCoord(t % tiles, tilesM, tilesN, groupN);
            const int rowA = tc.m * kCePairM + static_cast<int>(rank) * 128;
            const int rowB = tc.n * kCeAccN + static_cast<int>(rank) * 128;
            const int kBegin = t / tiles * kPerSplit, kEnd = min(numK, kBegin + kPerSplit);
            for (int kb = kBegin; kb < kEnd; ++kb) {
                if (!warp_all(mbar_wait(&emptyBar[stage], phase ^ 1u, abortFlag, status, kDevTimeoutStageEmpty))) {
                    alive = false;
                    break;
                }
                if (elect_one()) {
                    uint8_t* sa = smem + stage * kCeStageBytes;
                    uint8_t* sb = sa + kCeOperandBytes;
                    if (leader) mbar_arrive_expect_tx(&fullBar[stage], 2 * kCeStageBytes);
                    const uint32_t fullLeader = mapa_cluster(smem_u32(&fullBar[stage]), 0);
                    // K-major: one box of 128 rows x 64 k. MN-major: two boxes of 64 k-rows x 64 columns, 8 KiB each
                    if constexpr (kAMn) {
                        tma_load_2d_pair(sa, &tmapA, fullLeader, rowA, kb * kCeBlockK);
                        tma_load_2d_pair(sa + kCeOperandBytes / 2, &tmapA, fullLeader, rowA + 64, kb * kCeBlockK);
                    } else {
                        tma_load_2d_pair(sa, &tmapA, fullLeader, kb * kCeBlockK, rowA);
                    }
                    if constexpr (kBMn) {
                        tma_load_2d_pair(sb, &tmapB, fullLeader, rowB, kb * kCeBlockK);
                        tma_load_2d_pair(sb + kCeOperandBytes / 2, &tmapB, fullLeader, rowB + 64, kb * kCeBlockK);
                    } else {
                        tma_load_2d_pair(sb, &tmapB, fullLeader, kb * kCeBlockK, rowB);
                    }
                }
                __syncwarp();
                if (++stage == kCeStages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        }
    } else if (warp == 1 && leader) {
        // ---------------- MMA issuer (leader CTA only, one elected thread) ----------------
        if (elect_one()) {
            // K-major: 8-row groups 1024 B apart, 16 k are 32 B along a row. MN-major: 8-k groups 1024 B apart, 64-wide
            // slices half an operand apart, 16 k are 16 rows of 128 B.
            constexpr uint32_t kHi = smem_desc_hi_sw128(1024);
            constexpr uint32_t kStepA = (kAMn ? 16 * kCeRowBytes : 32) >> 4;
            constexpr uint32_t kStepB = (kBMn ? 16 * kCeRowBytes : 32) >> 4;
            const uint32_t a0 = smem_desc_lo(smem_u32(smem), kAMn ? kCeOperandBytes / 2 : 0);
            const uint32_t b0 = smem_desc_lo(smem_u32(smem) + kCeOperandBytes, kBMn ? kCeOperandBytes / 2 : 0);
            int stage = 0;
            uint32_t phase = 0;
            int local = 0;
            bool alive = true;
            for (int t = clusterId; t < totalTiles && alive; t += numClusters, ++local) {
                const int buf = local & 1;
                const uint32_t accPhase = static_cast<uint32_t>(local >> 1) & 1u;
                if (!mbar_wait(&accEmptyBar[buf], accPhase ^ 1u, abortFlag, status, kDevTimeoutAccEmpty)) break;
                tc_fence_after();
                const uint32_t dTmem = tmemBase + static_cast<uint32_t>(buf * kCeAccN);
                const int kBegin = t / tiles * kPerSplit, kEnd = min(numK, kBegin + kPerSplit);
                for (int kb = kBegin; kb < kEnd; ++kb) {
                    if (!mbar_wait(&fullBar[stage], phase, abortFlag, status, kDevTimeoutTmaFull)) {
                        alive = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t offset = static_cast<uint32_t>(stage) * (kCeStageBytes >> 4);
#pragma unroll
                    for (int kk = 0; kk < kCeBlockK / 16; ++kk) {
                        umma_f16_pair_words(dTmem, a0 + offset + kk * kStepA, kHi, b0 + offset + kk * kStepB, kHi, kIdesc,
                                            (kb > kBegin || kk > 0) ? 1u : 0u);
                    }
                    umma_commit_pair(&emptyBar[stage]);
                    if (kb == kEnd - 1) umma_commit_pair(&accFullBar[buf]);
                    if (++stage == kCeStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
        }
        __syncwarp();
    } else if (warp >= 4) {
        // ---------------- epilogue (both CTAs, 8 warps: lane quarter x column half) ----------------
        const int quarter = warp & 3;
        const int colHalf = (warp - 4) >> 2;
        uint8_t* stageTile = smem + kCeStages * kCeStageBytes + 256 + (warp - 4) * 4096;
        int local = 0;
        for (int t = clusterId; t < totalTiles; t += numClusters, ++local) {
            const CeTile tc = ceTileCoord(t % tiles, tilesM, tilesN, groupN);
            const int buf = local & 1;
            const uint32_t accPhase = static_cast<uint32_t>(local >> 1) & 1u;
            if (!warp_all(mbar_wait(&accFullBar[buf], accPhase, abortFlag, status, kDevTimeoutAccFull))) break;
            tc_fence_after();
            const int row0 = tc.m * kCePairM + static_cast<int>(rank) * 128 + quarter * 32;
            const int row = row0 + lane;
            const bool rowOk = row < m;
            const int firstCol = tc.n * kCeAccN + colHalf * 128;
            const uint32_t tBase = tmemBase + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(buf * kCeAccN + colHalf * 128);

            if constexpr (kMode == kCeStats) {
                const int64_t label = rowOk ? ceLabel(ep.labels[row], ep.vocab) - ep.firstColumn : -1;
                float top = -INFINITY, sum = 0.0f;
#pragma unroll 1
                for (int c = 0; c < 128; c += 32) {
                    const int col = firstCol + c;
                    if (col >= n) break;
                    uint32_t raw[32];
                    tmem_ld_32x32(tBase + static_cast<uint32_t>(c), raw);
                    tmem_ld_wait();
                    float v[32];
                    ceLogits(raw, v, ep.bias, col, n, lane);
                    ceAccumulate(v, top, sum);
                    if (label >= col && label < col + 32) {
                        float z = 0.0f;
#pragma unroll
                        for (int j = 0; j < 32; ++j) z = label == col + j ? v[j] : z;
                        ep.labelLogit[row] = z;
                    }
                }
                if (rowOk && firstCol < n) ep.partials[static_cast<size_t>(firstCol >> 7) * static_cast<size_t>(m) + row] = make_float2(top, sum);
            } else if constexpr (kMode == kCeDz) {
                float g = 0.0f, lse = 0.0f;
                int64_t label = -1;
                if (rowOk) {
                    label = ceLabel(ep.labels[row], ep.vocab);
                    if (label >= 0) g = ep.gradLoss != nullptr ? ep.gradLoss[row] : 1.0f;
                    label -= ep.firstColumn;
                    lse = ep.lse[row];
                }
                const int ld = static_cast<int>(ep.ldDz);
#pragma unroll 1
                for (int round = 0; round < 2; ++round) {   // 64 bf16 columns (one 128-byte line per row) per round
#pragma unroll
                    for (int sub = 0; sub < 2; ++sub) {
                        const int c = round * 64 + sub * 32;
                        const int col = firstCol + c;
                        uint32_t raw[32];
                        tmem_ld_32x32(tBase + static_cast<uint32_t>(c), raw);
                        tmem_ld_wait();
                        float v[32];
                        ceLogits(raw, v, ep.bias, col, n, lane);
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] = exp2f((v[j] - lse) * kLog2e);
                        if (label >= col && label < col + 32) {
#pragma unroll
                            for (int j = 0; j < 32; ++j) v[j] -= label == col + j ? 1.0f : 0.0f;
                        }
                        // a row that does not count is zero whatever its logits hold
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] = g != 0.0f ? v[j] * g : 0.0f;
#pragma unroll
                        for (int p = 0; p < 4; ++p) {
                            uint4 packed;
                            uint32_t* pw = reinterpret_cast<uint32_t*>(&packed);
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                // dz is the operand of two bf16 products: rounded once, here
                                const __nv_bfloat162 h = __floats2bfloat162_rn(v[p * 8 + 2 * j], v[p * 8 + 2 * j + 1]);
                                pw[j] = *reinterpret_cast<const uint32_t*>(&h);
                            }
                            *reinterpret_cast<uint4*>(stageTile + lane * 128 + (((sub * 4 + p) ^ (lane & 7)) << 4)) = packed;
                        }
                        if (ep.biasPartials != nullptr && row0 < m) {
                            const float total = warpColumnSums(v, lane);
                            ep.biasPartials[static_cast<size_t>(row0 >> 5) * static_cast<size_t>(ld) + col + lane] = total;
                        }
                    }
                    __syncwarp();
                    const int piece = lane & 7;
                    const int colOut = firstCol + round * 64 + piece * 8;   // the piece is padded to whole tiles: always inside
#pragma unroll
                    for (int q4 = 0; q4 < 8; ++q4) {
                        const int rr = q4 * 4 + (lane >> 3);
                        const uint4 val = *reinterpret_cast<const uint4*>(stageTile + rr * 128 + ((piece ^ (rr & 7)) << 4));
                        if (row0 + rr < m) *reinterpret_cast<uint4*>(ep.dz + static_cast<size_t>(row0 + rr) * static_cast<size_t>(ld) + colOut) = val;
                    }
                    __syncwarp();
                }
            } else {
                const float scale = ceScale(ep.dGradScale, ep.gradScale);   // the factor dz left out
                constexpr int kRoundCols = 128 / static_cast<int>(sizeof(TC));
                constexpr int kPieceCols = 16 / static_cast<int>(sizeof(TC));
                // a part of a split reduction goes to its own [m][ldOut] block
                TC* out = static_cast<TC*>(ep.out) + static_cast<size_t>(t / tiles) * static_cast<size_t>(m) * static_cast<size_t>(ep.ldOut);
#pragma unroll 1
                for (int round = 0; round < 128 / kRoundCols; ++round) {
                    const int col0 = firstCol + round * kRoundCols;
                    if (col0 >= n) break;
#pragma unroll
                    for (int sub = 0; sub < kRoundCols / 32; ++sub) {
                        uint32_t raw[32];
                        tmem_ld_32x32(tBase + static_cast<uint32_t>(round * kRoundCols + sub * 32), raw);
                        tmem_ld_wait();
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            const int col = col0 + sub * 32 + g * 8;
                            float v[8];
#pragma unroll
                            for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(raw[g * 8 + j]) * scale;
                            if (ep.addend != nullptr && rowOk && col + 8 <= n) {
                                const float4* r = reinterpret_cast<const float4*>(ep.addend + static_cast<size_t>(row) * static_cast<size_t>(ep.ldAddend) + col);
                                const float4 r0 = r[0], r1 = r[1];
                                v[0] += r0.x; v[1] += r0.y; v[2] += r0.z; v[3] += r0.w;
                                v[4] += r1.x; v[5] += r1.y; v[6] += r1.z; v[7] += r1.w;
                            }
                            if constexpr (sizeof(TC) == 4) {
                                *reinterpret_cast<float4*>(stageTile + lane * 128 + (((2 * g) ^ (lane & 7)) << 4)) = make_float4(v[0], v[1], v[2], v[3]);
                                *reinterpret_cast<float4*>(stageTile + lane * 128 + (((2 * g + 1) ^ (lane & 7)) << 4)) = make_float4(v[4], v[5], v[6], v[7]);
                            } else {
                                uint4 packed;
                                uint32_t* pw = reinterpret_cast<uint32_t*>(&packed);
#pragma unroll
                                for (int j = 0; j < 4; ++j) {
                                    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
                                    pw[j] = *reinterpret_cast<const uint32_t*>(&h);
                                }
                                *reinterpret_cast<uint4*>(stageTile + lane * 128 + (((sub * 4 + g) ^ (lane & 7)) << 4)) = packed;
                            }
                        }
                    }
                    __syncwarp();
                    const int piece = lane & 7;
                    const int colOut = col0 + piece * kPieceCols;
#pragma unroll
                    for (int q4 = 0; q4 < 8; ++q4) {
                        const int rr = q4 * 4 + (lane >> 3);
                        const uint4 val = *reinterpret_cast<const uint4*>(stageTile + rr * 128 + ((piece ^ (rr & 7)) << 4));
                        if (row0 + rr < m && colOut + kPieceCols <= n)
                            *reinterpret_cast<uint4*>(out + static_cast<size_t>(row0 + rr) * static_cast<size_t>(ep.ldOut) + colOut) = val;
                    }
                    __syncwarp();
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(mapa_cluster(smem_u32(&accEmptyBar[buf]), 0));
        }
    }

    // ---------------- teardown ----------------
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();  // the peer's shared and tensor memory stay alive until the leader's MMAs are done with them
    if (warp == 2) {
        if (*abortFlag != 0) {
            const uint64_t t0 = global_timer_ns();
            while (global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
        }
        tc_fence_after();
        tmem_dealloc(tmemBase, 512);
    }
}

// Operand [rows, cols] of bf16 with row pitch ld: K-major (rows are M or N, boxes of 128 rows x 64 k) or MN-major (rows
// are the reduction, boxes of 64 k x 64 columns).
void ceOperandMap(TensorMapStorage* out, const void* base, int64_t rows, int64_t cols, int64_t ld, bool mnMajor) {
    const uint64_t dims[2] = {static_cast<uint64_t>(cols), static_cast<uint64_t>(rows)};
    const uint64_t strides[1] = {static_cast<uint64_t>(ld) * 2};
    const uint32_t box[2] = {64u, mnMajor ? 64u : 128u};
    encodeTensorMap(out, base, 2, 2, dims, strides, box);
}

template <int kMode, bool kAMn, bool kBMn, typename TC>
void launchCe(const TensorMapStorage& ta, const TensorMapStorage& tb, const CeEpilogue& ep, int64_t m, int64_t n, int64_t k, int splits,
              int* status, cudaStream_t stream) {
    const int tilesM = static_cast<int>((m + kCePairM - 1) / kCePairM);
    const int tilesN = static_cast<int>((n + kCeAccN - 1) / kCeAccN);
    // about 4096 columns of B stay L2-resident while the rows sweep past (16 MB at a depth of 2048)
    const int groups = (tilesN + 15) / 16;
    const int groupN = (tilesN + groups - 1) / groups;
    const int stages = static_cast<int>((k + kCeBlockK - 1) / kCeBlockK);
    const int kPerSplit = (stages + splits - 1) / splits;
    splits = (stages + kPerSplit - 1) / kPerSplit;   // callers sized for this many parts (ceSplits)
    const int clusters = std::max(1, std::min(tilesM * tilesN * splits, persistentSms() / 2));
    auto kernel = cePairKernel<kMode, kAMn, kBMn, TC>;
    BFB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kCeSmemBytes));
    ProfileScope prof(kProfGemmTc, stream, 2.0 * static_cast<double>(m) * static_cast<double>(n) * static_cast<double>(k));
    launchDependent(kernel, dim3(2 * clusters), dim3(kCeThreads), kCeSmemBytes, stream, *reinterpret_cast<const CUtensorMap*>(ta.bytes),
                    *reinterpret_cast<const CUtensorMap*>(tb.bytes), ep, static_cast<int>(m), static_cast<int>(n), static_cast<int>(k), tilesM,
                    tilesN, groupN, kPerSplit, splits, status);
    BFB_LAUNCH_CHECK();
    noteLaunch();
}

}  // namespace

void ceStatsTensorCore(const LinearCeArgs& a, float2* partials, float* labelLogit, cudaStream_t stream) {
    TensorMapStorage tx, tw;
    ceOperandMap(&tx, a.x, a.tokens, a.dim, a.ldX, false);
    ceOperandMap(&tw, a.w, a.vocab, a.dim, a.ldW, false);
    CeEpilogue ep;
    ep.bias = a.bias;
    ep.labels = a.labels;
    ep.vocab = a.vocab;
    ep.partials = partials;
    ep.labelLogit = labelLogit;
    launchCe<kCeStats, false, false, float>(tx, tw, ep, a.tokens, a.vocab, a.dim, 1, a.dStatus, stream);
}

void ceDzTensorCore(const LinearCeArgs& a, int64_t firstColumn, int64_t columns, void* dz, int64_t ldDz, float* biasPartials,
                    cudaStream_t stream) {
    TensorMapStorage tx, tw;
    ceOperandMap(&tx, a.x, a.tokens, a.dim, a.ldX, false);
    ceOperandMap(&tw, static_cast<const __nv_bfloat16*>(a.w) + firstColumn * a.ldW, columns, a.dim, a.ldW, false);
    CeEpilogue ep;
    ep.bias = a.bias == nullptr ? nullptr : a.bias + firstColumn;
    ep.labels = a.labels;
    ep.vocab = a.vocab;
    ep.firstColumn = firstColumn;
    ep.lse = a.lseIn;
    ep.gradLoss = a.gradLoss;
    ep.dz = static_cast<__nv_bfloat16*>(dz);
    ep.ldDz = ldDz;
    ep.biasPartials = biasPartials;
    launchCe<kCeDz, false, false, float>(tx, tw, ep, a.tokens, columns, a.dim, 1, a.dStatus, stream);
}

int ceSplits(int64_t m, int64_t n, int64_t k) {
    const int64_t tiles = ((m + kCePairM - 1) / kCePairM) * ((n + kCeAccN - 1) / kCeAccN);
    const int64_t stages = (k + kCeBlockK - 1) / kCeBlockK;
    // 74 pairs whatever the device has free: the split decides how sums are grouped, and results do not depend on that.
    // Measured with 28 tiles over 782 stages (1543 x 1000 from 50021 columns): one part 271 us, five 125 + 13 us for their sum.
    // With more tiles than pairs only the last wave gains, less than the parts cost: 256 tiles in two parts took 16384 x 32000
    // x 2048 from 6.71 to 6.86 ms a step.
    constexpr int64_t kPairs = 74;
    if (tiles >= kPairs) return 1;
    int best = 1;
    double cost = static_cast<double>((tiles + kPairs - 1) / kPairs);
    for (int s = 2; s <= 16 && stages / s >= 16; ++s) {
        const double c = static_cast<double>((tiles * s + kPairs - 1) / kPairs) / s;
        if (c < 0.9 * cost) {
            best = s;
            cost = c;
        }
    }
    const int64_t per = (stages + best - 1) / best;
    return static_cast<int>((stages + per - 1) / per);
}

void ceDxTensorCore(const LinearCeArgs& a, int64_t firstColumn, int64_t columns, const void* dz, int64_t ldDz, void* out, int outDtype,
                    int64_t ldOut, const float* addend, int64_t ldAddend, int splits, cudaStream_t stream) {
    TensorMapStorage tz, tw;
    ceOperandMap(&tz, dz, a.tokens, columns, ldDz, false);
    ceOperandMap(&tw, static_cast<const __nv_bfloat16*>(a.w) + firstColumn * a.ldW, columns, a.dim, a.ldW, true);
    CeEpilogue ep;
    ep.dGradScale = a.dGradScale;
    ep.gradScale = a.gradScale;
    ep.out = out;
    ep.ldOut = ldOut;
    ep.addend = addend;
    ep.ldAddend = ldAddend;
    if (outDtype == BFB_F32) launchCe<kCeGrad, false, true, float>(tz, tw, ep, a.tokens, a.dim, columns, splits, a.dStatus, stream);
    else launchCe<kCeGrad, false, true, __nv_bfloat16>(tz, tw, ep, a.tokens, a.dim, columns, splits, a.dStatus, stream);
}

void ceDwTensorCore(const LinearCeArgs& a, int64_t columns, const void* dz, int64_t ldDz, void* out, int outDtype, int64_t ldOut, int splits,
                    cudaStream_t stream) {
    TensorMapStorage tz, tx;
    ceOperandMap(&tz, dz, a.tokens, columns, ldDz, true);
    ceOperandMap(&tx, a.x, a.tokens, a.dim, a.ldX, true);
    CeEpilogue ep;
    ep.dGradScale = a.dGradScale;
    ep.gradScale = a.gradScale;
    ep.out = out;
    ep.ldOut = ldOut;
    if (outDtype == BFB_F32) launchCe<kCeGrad, true, true, float>(tz, tx, ep, columns, a.dim, a.tokens, splits, a.dStatus, stream);
    else launchCe<kCeGrad, true, true, __nv_bfloat16>(tz, tx, ep, columns, a.dim, a.tokens, splits, a.dStatus, stream);
}

}  // namespace bfb
