// Softmax cross entropy of an output projection, without keeping the logits:
//
//   z = x W^T + b                       [tokens, vocab], never in memory as a whole
//   lse_t  = log sum_v exp z_tv,        loss_t = lse_t - z_t,label(t)
//   dz_tv  = g_t (exp(z_tv - lse_t) - [v = label(t)])
//   dx = dz W,  dW = dz^T x,  db = sum_t dz_t
//
// Forward: one product over all columns whose epilogue leaves a running maximum and a sum of exponentials per row and
// block of columns; a small kernel joins them. Backward: the vocabulary goes by in pieces; each piece's logits are
// computed again, become dz in the epilogue, and are used up by the two gradient products before the next piece
// overwrites them. That costs a fourth product (8 instead of 6 tokens x vocab x dim FLOPs with the gradient) and saves
// tokens x vocab words: 4.2 GB for 32 768 tokens and 32 000 classes.
//
// bf16 operands on 16-byte rows run on the tensor cores (linear_ce_tc.cu). fp32 operands, where products in fp32 are
// the contract, and bf16 rows that TMA cannot read run on the CUDA-core kernel below: 64 x 64 tiles, 4 x 4 per thread,
// the same two epilogues, dz kept in fp32. A gradient product with few tiles and a long reduction is split over it on both
// routes; the parts are added in order.
#include <cuda_bf16.h>

#include <algorithm>
#include <climits>

#include "common.cuh"
#include "kernels.hpp"
#include "linear_ce.cuh"
#include "ptx_sm100.cuh"

namespace bfb {

namespace {

constexpr int64_t kCeDzBytes = 256ll << 20;   // target size of one piece's dz
constexpr int kStatsColumnsTc = 128;          // columns behind one (maximum, sum) pair
constexpr int kStatsColumnsSimt = 64;

inline int64_t roundUp(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
inline bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// ---- CUDA-core products -----------------------------------------------------------------------------------

constexpr int kTile = 64, kDepth = 32;

template <typename T>
__device__ __forceinline__ float ceLoad(const void* p, int64_t i);
template <>
__device__ __forceinline__ float ceLoad<float>(const void* p, int64_t i) { return static_cast<const float*>(p)[i]; }
template <>
__device__ __forceinline__ float ceLoad<__nv_bfloat16>(const void* p, int64_t i) {
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

struct CeSimtArgs {
    const void* a;              // A(i, k) = a[i * aRow + k * aDepth]
    const void* b;              // B(k, j) = b[j * bRow + k * bDepth]
    int64_t aRow, aDepth, bRow, bDepth;
    int64_t m, n, k;
    // statistics, dz
    const float* bias;
    const float* labels;
    int64_t vocab, firstColumn;
    float2* partials;           // [parts][m]
    float* labelLogit;
    const float* lse;
    const float* gradLoss;
    const float* dGradScale;
    float gradScale;
    float* dz;                  // [m][ldDz]
    int64_t ldDz;
    // gradients
    void* out;
    int64_t ldOut;
    const float* addend;        // fp32 [m][ldAddend] or null
    int64_t ldAddend;
    int64_t kPerSplit;          // part of the reduction per blockIdx.y; parts go to [split][m][ldOut]
};

enum { kSimtStats = 0, kSimtDz = 1, kSimtGrad = 2 };

// The next slice of the operands is on its way to registers while this one is used: at these sizes a slice costs a trip to
// memory, not its arithmetic.
template <int kMode, typename TA, typename TB, typename TC>
__global__ void __launch_bounds__(256, 2) ceSimtKernel(const CeSimtArgs p) {
    pdl_launch_dependents();
    pdl_wait();
    __shared__ alignas(16) float sa[kDepth][kTile + 4];
    __shared__ alignas(16) float sb[kDepth][kTile + 4];
    __shared__ float2 rowStat[kTile][16];
    constexpr int kEach = kTile * kDepth / 256;
    const int tid = threadIdx.x;
    const int tx = tid & 15, ty = tid >> 4;
    const int64_t tilesN = (p.n + kTile - 1) / kTile;
    const int64_t tilesM = (p.m + kTile - 1) / kTile;
    const int64_t kBegin = static_cast<int64_t>(blockIdx.y) * p.kPerSplit, kEnd = min(p.k, kBegin + p.kPerSplit);
    const bool aAlong = p.aDepth == 1, bAlong = p.bDepth == 1;   // neighbouring threads go where memory is contiguous
    for (int64_t tile = blockIdx.x; tile < tilesM * tilesN; tile += gridDim.x) {
        const int64_t m0 = (tile / tilesN) * kTile, n0 = (tile % tilesN) * kTile;
        float acc[4][4] = {};
        float ra[kEach], rb[kEach];
        auto fetch = [&](int64_t k0) {
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                const int i = tid + e * 256;
                const int r0 = aAlong ? i / kDepth : i % kTile, k1 = aAlong ? i % kDepth : i / kTile;
                const int r2 = bAlong ? i / kDepth : i % kTile, k3 = bAlong ? i % kDepth : i / kTile;
                ra[e] = m0 + r0 < p.m && k0 + k1 < kEnd ? ceLoad<TA>(p.a, (m0 + r0) * p.aRow + (k0 + k1) * p.aDepth) : 0.0f;
                rb[e] = n0 + r2 < p.n && k0 + k3 < kEnd ? ceLoad<TB>(p.b, (n0 + r2) * p.bRow + (k0 + k3) * p.bDepth) : 0.0f;
            }
        };
        fetch(kBegin);
        for (int64_t k0 = kBegin; k0 < kEnd; k0 += kDepth) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                const int i = tid + e * 256;
                if (aAlong) sa[i % kDepth][i / kDepth] = ra[e];
                else sa[i / kTile][i % kTile] = ra[e];
                if (bAlong) sb[i % kDepth][i / kDepth] = rb[e];
                else sb[i / kTile][i % kTile] = rb[e];
            }
            __syncthreads();
            if (k0 + kDepth < kEnd) fetch(k0 + kDepth);
#pragma unroll
            for (int kk = 0; kk < kDepth; ++kk) {
                const float4 a4 = *reinterpret_cast<const float4*>(&sa[kk][ty * 4]);
                const float4 b4 = *reinterpret_cast<const float4*>(&sb[kk][tx * 4]);
                const float av[4] = {a4.x, a4.y, a4.z, a4.w}, bv[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(av[i], bv[j], acc[i][j]);
            }
        }
        if constexpr (kMode == kSimtGrad) {
            TC* out = static_cast<TC*>(p.out) + static_cast<int64_t>(blockIdx.y) * p.m * p.ldOut;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int64_t row = m0 + ty * 4 + i;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int64_t col = n0 + tx * 4 + j;
                    if (row >= p.m || col >= p.n) continue;
                    float v = acc[i][j];
                    if (p.addend != nullptr) v += p.addend[row * p.ldAddend + col];
                    if constexpr (sizeof(TC) == 4) out[row * p.ldOut + col] = v;
                    else out[row * p.ldOut + col] = __float2bfloat16_rn(v);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t col = n0 + tx * 4 + j;
                const float b = col >= p.n ? -INFINITY : (p.bias != nullptr ? p.bias[col] : 0.0f);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[i][j] += b;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int64_t row = m0 + ty * 4 + i;
                if (row >= p.m) continue;
                const int64_t label = ceLabel(p.labels[row], p.vocab);
                if constexpr (kMode == kSimtStats) {
                    float top = -INFINITY, sum = 0.0f;
                    ceAccumulate(acc[i], top, sum);
                    rowStat[ty * 4 + i][tx] = make_float2(top, sum);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (label >= 0 && label - p.firstColumn == n0 + tx * 4 + j) p.labelLogit[row] = acc[i][j];
                } else {
                    const float g = label >= 0 ? ceRowGrad(p.gradLoss, row, p.dGradScale, p.gradScale) : 0.0f;
                    const float lse = p.lse[row];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int64_t col = n0 + tx * 4 + j;
                        if (col >= p.n) continue;
                        float v = exp2f((acc[i][j] - lse) * kLog2e);
                        if (label - p.firstColumn == col) v -= 1.0f;
                        p.dz[row * p.ldDz + col] = g != 0.0f ? v * g : 0.0f;   // a row that does not count is zero whatever its logits hold
                    }
                }
            }
            if constexpr (kMode == kSimtStats) {
                __syncthreads();
                if (tid < kTile && m0 + tid < p.m) {
                    float top = rowStat[tid][0].x;
                    for (int c = 1; c < 16; ++c) top = fmaxf(top, rowStat[tid][c].x);
                    const float at = top == -INFINITY ? 0.0f : top;
                    float sum = 0.0f;
                    for (int c = 0; c < 16; ++c) sum += rowStat[tid][c].y * exp2f((rowStat[tid][c].x - at) * kLog2e);
                    p.partials[(n0 / kTile) * p.m + m0 + tid] = make_float2(top, sum);
                }
            }
        }
    }
}

// ---- joining the pieces of the forward --------------------------------------------------------------------------

// 32 rows per block, the parts of a row split over the block's warps and joined through shared memory, in the same order on
// every run. A warp's parts come in batches of four.
__global__ void __launch_bounds__(1024)
ceFinishKernel(const float2* __restrict__ partials, int64_t parts, const float* __restrict__ labelLogit, const float* __restrict__ labels,
               int64_t vocab, float* loss, float* lse, int64_t tokens, int* oobCount) {
    pdl_launch_dependents();
    pdl_wait();
    __shared__ float2 joined[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    float top = -INFINITY, sum = 0.0f;
    auto join = [&](const float2& s) {
        const float next = fmaxf(top, s.x);
        const float at = next == -INFINITY ? 0.0f : next;
        sum = sum * exp2f((top - at) * kLog2e) + s.y * exp2f((s.x - at) * kLog2e);
        top = next;
    };
    if (row < tokens) {
        for (int64_t part = warp; part < parts; part += 4 * warps) {
            float2 s[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int64_t at = part + u * warps;
                s[u] = at < parts ? partials[at * tokens + row] : make_float2(-INFINITY, 0.0f);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) join(s[u]);
        }
    }
    joined[warp][lane] = make_float2(top, sum);
    __syncthreads();
    if (warp != 0 || row >= tokens) return;
    for (int w = 1; w < warps; ++w) join(joined[w][lane]);
    const float value = top + logf(sum);   // no column above -inf: -inf + log 0, a row without a distribution
    lse[row] = value;
    const float label = labels[row];
    const bool counted = ceLabel(label, vocab) >= 0;
    if (loss != nullptr) loss[row] = counted ? value - labelLogit[row] : 0.0f;
    if (oobCount != nullptr && ceLabelIsBad(label, vocab)) atomicAdd(oobCount, 1);
}

// {sum of the losses, rows that count, 1 / rows that count}: one block, a fixed order, the sum in 64 bits.
__global__ void __launch_bounds__(1024)
ceSummaryKernel(const float* __restrict__ loss, const float* __restrict__ labels, int64_t vocab, int64_t tokens, float* summary) {
    pdl_launch_dependents();
    pdl_wait();
    __shared__ double sums[32];
    __shared__ unsigned long long counts[32];
    double sum = 0.0;
    unsigned long long count = 0;
    for (int64_t i0 = threadIdx.x; i0 < tokens; i0 += 8 * 1024) {
        float label[8], value[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {   // all loads of a batch before its sums
            const int64_t i = min(i0 + u * 1024, tokens - 1);
            label[u] = labels[i];
            value[u] = loss[i];
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            if (i0 + u * 1024 < tokens && ceLabel(label[u], vocab) >= 0) {
                sum += value[u];
                ++count;
            }
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        count += __shfl_xor_sync(0xFFFFFFFFu, count, o);
    }
    if ((threadIdx.x & 31) == 0) {
        sums[threadIdx.x >> 5] = sum;
        counts[threadIdx.x >> 5] = count;
    }
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int w = 1; w < 32; ++w) {
        sum += sums[w];
        count += counts[w];
    }
    summary[0] = static_cast<float>(sum);
    summary[1] = static_cast<float>(count);
    summary[2] = count == 0 ? 0.0f : static_cast<float>(1.0 / static_cast<double>(count));
}

// Column sums of `rows` rows of partial sums (or of dz itself), times a factor: 32 columns per block, the rows split over eight warps.
__global__ void __launch_bounds__(256)
ceColumnSumKernel(const float* __restrict__ in, int64_t ld, int64_t rows, int64_t columns, const float* dScale, float scale, float* out) {
    pdl_launch_dependents();
    pdl_wait();
    __shared__ float joined[8][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t col = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    float sum = 0.0f;
    if (col < columns) {
        for (int64_t r = warp; r < rows; r += 8) sum += in[r * ld + col];
    }
    joined[warp][lane] = sum;
    __syncthreads();
    if (warp != 0 || col >= columns) return;
    for (int w = 1; w < 8; ++w) sum += joined[w][lane];
    out[col] = sum * ceScale(dScale, scale);
}

// out = sum of the parts of a split product, in order, + addend.
template <typename TC>
__global__ void __launch_bounds__(256)
cePartSumKernel(const float* __restrict__ parts, int splits, int64_t rows, int64_t cols, const float* addend, int64_t ldAddend, TC* out,
                int64_t ldOut) {
    pdl_launch_dependents();
    pdl_wait();
    const int64_t total = rows * cols, step = static_cast<int64_t>(gridDim.x) * blockDim.x;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += step) {
        const int64_t row = i / cols, col = i - row * cols;
        float sum = parts[i];
        for (int s0 = 1; s0 < splits; s0 += 4) {
            float v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = s0 + u < splits ? parts[(s0 + u) * total + i] : 0.0f;
#pragma unroll
            for (int u = 0; u < 4; ++u) sum += v[u];
        }
        if (addend != nullptr) sum += addend[row * ldAddend + col];
        if constexpr (sizeof(TC) == 4) out[row * ldOut + col] = sum;
        else out[row * ldOut + col] = __float2bfloat16_rn(sum);
    }
}

void cePartSum(const float* parts, int splits, int64_t rows, int64_t cols, const float* addend, int64_t ldAddend, void* out, int outDtype,
               int64_t ldOut, cudaStream_t stream) {
    const int grid = static_cast<int>(std::min<int64_t>((rows * cols + 255) / 256, static_cast<int64_t>(smCount()) * 16));
    if (outDtype == BFB_F32) launchDependent(cePartSumKernel<float>, dim3(grid), dim3(256), 0, stream, parts, splits, rows, cols, addend, ldAddend, static_cast<float*>(out), ldOut);
    else launchDependent(cePartSumKernel<__nv_bfloat16>, dim3(grid), dim3(256), 0, stream, parts, splits, rows, cols, addend, ldAddend, static_cast<__nv_bfloat16*>(out), ldOut);
    BFB_LAUNCH_CHECK();
    noteLaunch();
}

__global__ void ceZeroRowsKernel(void* out, int dtype, int64_t ld, int64_t rows, int64_t cols) {
    const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < rows * cols; i += step) {
        const int64_t at = i / cols * ld + i % cols;
        if (dtype == BFB_F32) static_cast<float*>(out)[at] = 0.0f;
        else static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(0.0f);
    }
}

int simtGrid(int64_t m, int64_t n) {
    const int64_t tiles = ((m + kTile - 1) / kTile) * ((n + kTile - 1) / kTile);
    return static_cast<int>(std::min<int64_t>(tiles, static_cast<int64_t>(smCount()) * 8));
}

CeSimtArgs simtOperands(const LinearCeArgs& a, int64_t firstColumn, int64_t columns) {
    CeSimtArgs p{};
    p.a = a.x;
    p.aRow = a.ldX;
    p.aDepth = 1;
    p.b = a.dtype == BFB_F32 ? static_cast<const void*>(static_cast<const float*>(a.w) + firstColumn * a.ldW)
                             : static_cast<const void*>(static_cast<const __nv_bfloat16*>(a.w) + firstColumn * a.ldW);
    p.bRow = a.ldW;
    p.bDepth = 1;
    p.m = a.tokens;
    p.n = columns;
    p.k = a.dim;
    p.kPerSplit = a.dim;
    p.bias = a.bias == nullptr ? nullptr : a.bias + firstColumn;
    p.labels = a.labels;
    p.vocab = a.vocab;
    p.firstColumn = firstColumn;
    return p;
}

// ---- sizes ------------------------------------------------------------------------------------------------------

struct CePlan {
    bool tensorCores = false;
    int64_t parts = 0;          // (maximum, sum) pairs per row
    int64_t pieceColumns = 0;   // vocabulary columns per piece of the backward
    int64_t pieces = 0;
    int64_t ldDz = 0;
    int splitsDx = 1, splitsDw = 1;
    size_t forwardBytes = 0, dzBytes = 0, biasBytes = 0, dxBytes = 0, partBytes = 0;
    size_t backwardBytes() const { return dzBytes + biasBytes + dxBytes + partBytes; }
};

// The CUDA-core products: parts of at least 64 until there are two blocks for each of 148 SMs.
int simtSplits(int64_t m, int64_t n, int64_t k) {
    const int64_t tiles = ((m + kTile - 1) / kTile) * ((n + kTile - 1) / kTile);
    const int64_t want = std::max<int64_t>(1, std::min((2 * 148 + tiles - 1) / tiles, (k + 63) / 64));
    const int64_t per = (k + want - 1) / want;
    return static_cast<int>((k + per - 1) / per);
}

// The piece is as wide as its dz stays within 256 MiB, at least 4096 columns (narrower pieces make the dx product so
// shallow that the fp32 sums it carries from piece to piece cost more than its MMAs).
CePlan cePlan(int64_t tokens, int64_t vocab, int64_t dim, bool tensorCores) {
    CePlan p;
    p.tensorCores = tensorCores;
    const int64_t elem = tensorCores ? 2 : 4;
    const int64_t tile = tensorCores ? 256 : kTile;
    const int64_t part = tensorCores ? kStatsColumnsTc : kStatsColumnsSimt;
    p.parts = (vocab + part - 1) / part;
    const int64_t rows = std::max<int64_t>(tokens, 1);
    const int64_t widest = std::max<int64_t>(4096, kCeDzBytes / (elem * rows) / tile * tile);
    const int64_t vocabTiles = (vocab + tile - 1) / tile;
    int64_t width = std::min(widest / tile, vocabTiles);
    if (tensorCores && width < vocabTiles) {
        // dW's tiles of a piece go over 74 CTA pairs in waves, and a last wave that is nearly empty costs as much as a full
        // one: of the widths down to half the widest, the one with the fewest waves in all (a quarter of a wave for a piece more)
        const int64_t across = (dim + 255) / 256;
        auto waves = [&](int64_t w) {
            const int64_t whole = vocabTiles / w, rest = vocabTiles % w;
            return static_cast<double>(whole * ((w * across + 73) / 74) + (rest * across + 73) / 74) + 0.25 * static_cast<double>(whole + (rest > 0));
        };
        const int64_t most = width;
        for (int64_t w = most - 1; w >= (most + 1) / 2; --w)
            if (waves(w) < waves(width)) width = w;
    }
    p.pieceColumns = width * tile;
    p.pieces = (vocab + p.pieceColumns - 1) / p.pieceColumns;
    p.ldDz = p.pieceColumns;
    p.forwardBytes = static_cast<size_t>(roundUp(p.parts * rows * 8, 256) + roundUp(rows * 4, 256));
    p.dzBytes = static_cast<size_t>(roundUp(rows * p.ldDz * elem, 256));
    p.biasBytes = tensorCores ? static_cast<size_t>(roundUp((rows + 31) / 32 * p.ldDz * 4, 256)) : 0;
    p.dxBytes = p.pieces > 1 ? static_cast<size_t>(roundUp(rows * dim * 4, 256)) : 0;
    // all pieces alike, the narrower last one too
    p.splitsDx = tensorCores ? ceSplits(rows, dim, p.pieceColumns) : simtSplits(rows, dim, p.pieceColumns);
    p.splitsDw = tensorCores ? ceSplits(p.pieceColumns, dim, rows) : simtSplits(p.pieceColumns, dim, rows);
    const int64_t partsDx = p.splitsDx > 1 ? p.splitsDx * rows * dim : 0, partsDw = p.splitsDw > 1 ? p.splitsDw * p.pieceColumns * dim : 0;
    p.partBytes = static_cast<size_t>(roundUp(std::max(partsDx, partsDw) * 4, 256));
    return p;
}

void checkCommon(const LinearCeArgs& a, const char* what) {
    const std::string name = std::string("linear_cross_entropy_") + what + ": ";
    auto need = [&](bool ok, const char* text) { if (!ok) fail(BFB_INVALID_ARGUMENT, name + text); };
    need(a.dtype == BFB_F32 || a.dtype == BFB_BF16, "operands must be f32 or bf16");
    need(a.tokens >= 0 && a.vocab > 0 && a.dim > 0, "sizes must be positive");
    need(a.tokens < (1ll << 31) - 256 && a.vocab <= (1ll << 24) && a.dim < (1ll << 31) - 256, "sizes beyond the limits (2^31 rows, 2^24 classes)");
    need(a.ldX >= a.dim && a.ldW >= a.dim, "row pitch smaller than dim");
    need(a.tokens == 0 || (a.x != nullptr && a.labels != nullptr), "null pointer");
    need(a.w != nullptr, "null pointer");
}

void checkWorkspace(const LinearCeArgs& a, size_t need) {
    require(a.tokens == 0 || (a.workspace != nullptr && a.workspaceBytes >= need && reinterpret_cast<uintptr_t>(a.workspace) % 256 == 0),
            "linear_cross_entropy: the workspace is missing, too small (bfb_linear_cross_entropy_workspace) or not 256-byte aligned");
}

}  // namespace

size_t linearCeWorkspaceBytes(int dtype, int64_t tokens, int64_t vocab, int64_t dim, bool backward) {
    require(dtype == BFB_F32 || dtype == BFB_BF16, "linear_cross_entropy_workspace: operands must be f32 or bf16");
    require(tokens >= 0 && vocab > 0 && dim > 0, "linear_cross_entropy_workspace: sizes must be positive");
    require(tokens < (1ll << 31) - 256 && vocab <= (1ll << 24) && dim < (1ll << 31) - 256,
            "linear_cross_entropy_workspace: sizes beyond the limits (2^31 rows, 2^24 classes)");
    // pointers decide the route of a call, so the size covers both
    size_t most = 0;
    for (const bool tc : {false, true}) {
        if (tc && dtype != BFB_BF16) continue;
        const CePlan p = cePlan(tokens, vocab, dim, tc);
        most = std::max(most, p.forwardBytes);
        if (backward) most = std::max(most, p.backwardBytes());
    }
    return most;
}

bool linearCeUsesTensorCores(const LinearCeArgs& a) {
    return a.dtype == BFB_BF16 && a.dim % 8 == 0 && a.ldX % 8 == 0 && a.ldW % 8 == 0 && aligned16(a.x) && aligned16(a.w);
}

void linearCeForward(const LinearCeArgs& a, cudaStream_t stream) {
    checkCommon(a, "fwd");
    require(a.tokens == 0 || a.lse != nullptr, "linear_cross_entropy_fwd: null pointer");
    require(a.summary == nullptr || a.loss != nullptr, "linear_cross_entropy_fwd: the summary needs the losses");
    const bool tc = linearCeUsesTensorCores(a);
    const CePlan plan = cePlan(a.tokens, a.vocab, a.dim, tc);
    checkWorkspace(a, plan.forwardBytes);
    if (a.tokens > 0) {
        auto* base = static_cast<uint8_t*>(a.workspace);
        auto* partials = reinterpret_cast<float2*>(base);
        auto* labelLogit = reinterpret_cast<float*>(base + roundUp(plan.parts * a.tokens * 8, 256));
        if (tc) {
            ceStatsTensorCore(a, partials, labelLogit, stream);
        } else {
            CeSimtArgs p = simtOperands(a, 0, a.vocab);
            p.partials = partials;
            p.labelLogit = labelLogit;
            const int grid = simtGrid(p.m, p.n);
            if (a.dtype == BFB_F32) launchDependent(ceSimtKernel<kSimtStats, float, float, float>, dim3(grid), dim3(256), 0, stream, p);
            else launchDependent(ceSimtKernel<kSimtStats, __nv_bfloat16, __nv_bfloat16, float>, dim3(grid), dim3(256), 0, stream, p);
            BFB_LAUNCH_CHECK();
            noteLaunch();
        }
        // a warp of 32 rows for every four parts, up to 32 of them
        const int finishThreads = static_cast<int>(std::min<int64_t>(32, (plan.parts + 3) / 4)) * 32;
        launchDependent(ceFinishKernel, dim3(static_cast<unsigned>((a.tokens + 31) / 32)), dim3(finishThreads), 0, stream, partials, plan.parts, labelLogit, a.labels, a.vocab,
                                                                                      a.loss, a.lse, a.tokens, a.oobCount);
        BFB_LAUNCH_CHECK();
        noteLaunch();
    }
    if (a.summary != nullptr) {
        launchDependent(ceSummaryKernel, dim3(1), dim3(1024), 0, stream, a.loss, a.labels, a.vocab, a.tokens, a.summary);
        BFB_LAUNCH_CHECK();
        noteLaunch();
    }
}

void linearCeBackward(const LinearCeArgs& a, cudaStream_t stream) {
    checkCommon(a, "bwd");
    require(a.gradDtype == BFB_F32 || a.gradDtype == BFB_BF16, "linear_cross_entropy_bwd: gradients must be f32 or bf16");
    require(a.tokens == 0 || a.lseIn != nullptr, "linear_cross_entropy_bwd: null pointer");
    require((a.dx == nullptr || a.ldDx >= a.dim) && (a.dw == nullptr || a.ldDw >= a.dim), "linear_cross_entropy_bwd: row pitch smaller than dim");
    if (a.dx == nullptr && a.dw == nullptr && a.db == nullptr) return;
    const int64_t elem = a.gradDtype == BFB_F32 ? 4 : 2;
    auto vectorRows = [&](const void* p, int64_t ld) { return p == nullptr || (aligned16(p) && ld * elem % 16 == 0); };
    const bool tc = linearCeUsesTensorCores(a) && vectorRows(a.dx, a.ldDx) && vectorRows(a.dw, a.ldDw);
    const CePlan plan = cePlan(a.tokens, a.vocab, a.dim, tc);
    checkWorkspace(a, plan.backwardBytes());
    if (a.tokens == 0) {   // no rows: the sums over them are zero
        if (a.dw != nullptr) {
            ceZeroRowsKernel<<<smCount() * 4, 256, 0, stream>>>(a.dw, a.gradDtype, a.ldDw, a.vocab, a.dim);
            BFB_LAUNCH_CHECK();
            noteLaunch();
        }
        if (a.db != nullptr) BFB_CUDA(cudaMemsetAsync(a.db, 0, static_cast<size_t>(a.vocab) * 4, stream));
        return;
    }
    auto* base = static_cast<uint8_t*>(a.workspace);
    void* dz = base;
    auto* biasPartials = reinterpret_cast<float*>(base + plan.dzBytes);
    auto* dxSum = reinterpret_cast<float*>(base + plan.dzBytes + plan.biasBytes);
    auto* parts = reinterpret_cast<float*>(base + plan.dzBytes + plan.biasBytes + plan.dxBytes);
    const bool f32 = a.dtype == BFB_F32;
    auto simtProduct = [&](CeSimtArgs g, const void* b, bool bIsF32, int outDtype, int splits) {
        g.b = b;
        g.kPerSplit = (g.k + splits - 1) / splits;
        const dim3 grid(simtGrid(g.m, g.n), static_cast<unsigned>((g.k + g.kPerSplit - 1) / g.kPerSplit));
        if (bIsF32 && outDtype == BFB_F32) launchDependent(ceSimtKernel<kSimtGrad, float, float, float>, dim3(grid), dim3(256), 0, stream, g);
        else if (bIsF32) launchDependent(ceSimtKernel<kSimtGrad, float, float, __nv_bfloat16>, dim3(grid), dim3(256), 0, stream, g);
        else if (outDtype == BFB_F32) launchDependent(ceSimtKernel<kSimtGrad, float, __nv_bfloat16, float>, dim3(grid), dim3(256), 0, stream, g);
        else launchDependent(ceSimtKernel<kSimtGrad, float, __nv_bfloat16, __nv_bfloat16>, dim3(grid), dim3(256), 0, stream, g);
        BFB_LAUNCH_CHECK();
        noteLaunch();
        return static_cast<int>(grid.y);
    };
    auto partsOf = [](int64_t k, int splits, int64_t unit) {   // parts a product over k is really cut into
        const int64_t stages = (k + unit - 1) / unit, per = (stages + splits - 1) / splits;
        return static_cast<int>((stages + per - 1) / per);
    };
    for (int64_t piece = 0; piece < plan.pieces; ++piece) {
        const int64_t first = piece * plan.pieceColumns;
        const int64_t columns = std::min(plan.pieceColumns, a.vocab - first);
        const bool last = piece + 1 == plan.pieces;
        // dx: fp32 sums from piece to piece, the result's format with the last one
        const float* addend = piece == 0 ? nullptr : dxSum;
        void* dxOut = last ? a.dx : static_cast<void*>(dxSum);
        const int dxType = last ? a.gradDtype : BFB_F32;
        const int64_t ldDxOut = last ? a.ldDx : a.dim;
        void* dwOut = a.dw == nullptr ? nullptr : static_cast<uint8_t*>(a.dw) + first * a.ldDw * elem;
        const bool splitDx = plan.splitsDx > 1, splitDw = plan.splitsDw > 1;
        int partsDx = 1, partsDw = 1;
        if (tc) {
            ceDzTensorCore(a, first, columns, dz, plan.ldDz, a.db == nullptr ? nullptr : biasPartials, stream);
            if (a.dw != nullptr) {
                if (splitDw) {
                    ceDwTensorCore(a, columns, dz, plan.ldDz, parts, BFB_F32, a.dim, plan.splitsDw, stream);
                    partsDw = partsOf(a.tokens, plan.splitsDw, 64);
                } else {
                    ceDwTensorCore(a, columns, dz, plan.ldDz, dwOut, a.gradDtype, a.ldDw, 1, stream);
                }
            }
        } else {
            CeSimtArgs p = simtOperands(a, first, columns);
            p.lse = a.lseIn;
            p.gradLoss = a.gradLoss;
            p.dGradScale = a.dGradScale;
            p.gradScale = a.gradScale;
            p.dz = static_cast<float*>(dz);
            p.ldDz = plan.ldDz;
            if (f32) launchDependent(ceSimtKernel<kSimtDz, float, float, float>, dim3(simtGrid(p.m, p.n)), dim3(256), 0, stream, p);
            else launchDependent(ceSimtKernel<kSimtDz, __nv_bfloat16, __nv_bfloat16, float>, dim3(simtGrid(p.m, p.n)), dim3(256), 0, stream, p);
            BFB_LAUNCH_CHECK();
            noteLaunch();
            if (a.dw != nullptr) {   // dW(v, d) = sum_t dz(t, v) x(t, d)
                CeSimtArgs w{};
                w.a = dz;
                w.aRow = 1;
                w.aDepth = plan.ldDz;
                w.bRow = 1;
                w.bDepth = a.ldX;
                w.m = columns;
                w.n = a.dim;
                w.k = a.tokens;
                w.out = splitDw ? parts : dwOut;
                w.ldOut = splitDw ? a.dim : a.ldDw;
                partsDw = simtProduct(w, a.x, f32, splitDw ? BFB_F32 : a.gradDtype, plan.splitsDw);
            }
        }
        if (a.dw != nullptr && splitDw) cePartSum(parts, partsDw, columns, a.dim, nullptr, 0, dwOut, a.gradDtype, a.ldDw, stream);
        if (a.dx != nullptr) {   // dx(t, d) = sum_v dz(t, v) W(v, d)
            if (tc) {
                if (splitDx) ceDxTensorCore(a, first, columns, dz, plan.ldDz, parts, BFB_F32, a.dim, nullptr, 0, plan.splitsDx, stream);
                else ceDxTensorCore(a, first, columns, dz, plan.ldDz, dxOut, dxType, ldDxOut, addend, a.dim, 1, stream);
                partsDx = partsOf(columns, plan.splitsDx, 64);
            } else {
                CeSimtArgs x{};
                x.a = dz;
                x.aRow = plan.ldDz;
                x.aDepth = 1;
                x.bRow = 1;
                x.bDepth = a.ldW;
                x.m = a.tokens;
                x.n = a.dim;
                x.k = columns;
                x.out = splitDx ? parts : dxOut;
                x.ldOut = splitDx ? a.dim : ldDxOut;
                x.addend = splitDx ? nullptr : addend;
                x.ldAddend = a.dim;
                partsDx = simtProduct(x, simtOperands(a, first, columns).b, f32, splitDx ? BFB_F32 : dxType, plan.splitsDx);
            }
            if (splitDx) cePartSum(parts, partsDx, a.tokens, a.dim, addend, a.dim, dxOut, dxType, ldDxOut, stream);
        }
        if (a.db != nullptr) {
            const unsigned blocks = static_cast<unsigned>((columns + 31) / 32);
            if (tc) launchDependent(ceColumnSumKernel, dim3(blocks), dim3(256), 0, stream, biasPartials, plan.ldDz, (a.tokens + 31) / 32, columns, a.dGradScale, a.gradScale, a.db + first);
            else launchDependent(ceColumnSumKernel, dim3(blocks), dim3(256), 0, stream, static_cast<const float*>(dz), plan.ldDz, a.tokens, columns, nullptr, 1.0f, a.db + first);
            BFB_LAUNCH_CHECK();
            noteLaunch();
        }
    }
}

}  // namespace bfb
