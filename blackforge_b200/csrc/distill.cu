// Distillation from the top logits of a teacher: loss and gradient in one pass over the student's logits.
//
//   q = softmax(teacher / tau) over the listed entries,   p = softmax(z / tau) over the vocabulary
//   loss_t = tau^2 sum_k q_k (log q_k - log p_{i_k}),     dz_tj = g_t tau (p_tj - sum_{k: i_k = j} q_k)
//
// Bound by memory: the least a step can move is the logits once in and the gradient once out. So a row stays on the chip
// between the softmax statistics and the gradient: a cluster of up to eight blocks holds it in registers (16 bytes x
// kVecs a thread), every warp reduces its own maximum and sum, pushes the pair into the shared memory of all blocks of
// the cluster, and after one cluster barrier each warp joins all pairs in the same order and finishes its part of the
// row. Only what a row has beyond the capacity of a cluster is read again.
#include <cuda_bf16.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.hpp"
#include "linear_ce.cuh"
#include "ptx_sm100.cuh"

namespace bfb {

namespace {

constexpr int kMaxTeacher = 1024;
constexpr int kMaxCluster = 8;

// 16 bytes of a row: 4 fp32 or 8 bf16 values.
template <typename T>
struct RowVec {
    static constexpr int kN = 16 / static_cast<int>(sizeof(T));
};

__device__ __forceinline__ float distillToFloat(float v) { return v; }
__device__ __forceinline__ float distillToFloat(__nv_bfloat16 v) { return __bfloat162float(v); }

__device__ __forceinline__ void distillUnpack(const uint4& raw, float (&v)[4]) {
    v[0] = __uint_as_float(raw.x); v[1] = __uint_as_float(raw.y); v[2] = __uint_as_float(raw.z); v[3] = __uint_as_float(raw.w);
}
__device__ __forceinline__ void distillUnpack(const uint4& raw, float (&v)[8]) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        v[2 * j] = __uint_as_float(w[j] << 16);
        v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
    }
}

// Elements [first, first + kN) of a row of `count`; what lies outside reads as -inf. Whole vectors are 16-byte aligned.
template <typename T>
__device__ __forceinline__ uint4 distillLoad(const T* row, int first, int count) {
    constexpr int kN = RowVec<T>::kN;
    if (first >= 0 && first + kN <= count) return __ldcs(reinterpret_cast<const uint4*>(row + first));
    uint4 raw;
    T part[kN];
#pragma unroll
    for (int j = 0; j < kN; ++j) {
        const int at = first + j;
        if constexpr (sizeof(T) == 4) part[j] = at >= 0 && at < count ? row[at] : -INFINITY;
        else part[j] = at >= 0 && at < count ? row[at] : __ushort_as_bfloat16(0xFF80u);
    }
    __builtin_memcpy(&raw, part, 16);
    return raw;
}

// kN gradient values at `first` of a row; `aligned`: the row's whole vectors can be stored as such.
template <typename T, int kN>
__device__ __forceinline__ void distillStore(T* row, int first, int count, const float (&v)[kN], bool aligned) {
    if (aligned && first >= 0 && first + kN <= count) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < kN; j += 4)
                __stcs(reinterpret_cast<float4*>(row + first + j), make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]));
        } else {
            uint32_t w[kN / 2];
#pragma unroll
            for (int j = 0; j < kN / 2; ++j) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);   // the result's format: one rounding
                w[j] = *reinterpret_cast<const uint32_t*>(&h);
            }
            if constexpr (kN == 8) __stcs(reinterpret_cast<uint4*>(row + first), make_uint4(w[0], w[1], w[2], w[3]));
            else __stcs(reinterpret_cast<uint2*>(row + first), make_uint2(w[0], w[1]));
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < kN; ++j) {
        const int at = first + j;
        if (at < 0 || at >= count) continue;
        if constexpr (sizeof(T) == 4) row[at] = v[j];
        else row[at] = __float2bfloat16_rn(v[j]);
    }
}

struct DistillParams {
    const void* logits;
    int64_t ldLogits;
    const float* ids;        // [rows][k]
    const void* teacher;     // [rows][k], f32 or bf16
    int teacherBf16;
    int k;
    float tau;
    const float* gradLoss;
    const float* dGradScale;
    float gradScale;
    float* loss;
    float* lse;
    void* grad;              // may be the logits themselves
    int64_t ldGrad;
    int vocab;
    int* oobCount;
};

template <typename TIn, typename TOut, int kVecs, int kMaxThreads>
__global__ void __launch_bounds__(kMaxThreads)
distillKernel(const DistillParams p, int cluster) {
    constexpr int kN = RowVec<TIn>::kN;
    __shared__ float2 stats[kMaxCluster * 32];   // (maximum, sum) of every warp of the cluster, block by block
    __shared__ float teacherSum[2];              // teacher's sum of exponentials, its maximum
    extern __shared__ float dyn[];
    float* sQ = dyn;                             // [k]: teacher logit, then q
    float* sZ = dyn + p.k;                       // [k]: the student's logit at the entry
    int* sId = reinterpret_cast<int*>(dyn + 2 * p.k);

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
    const int rank = static_cast<int>(cluster_ctarank());
    const int64_t row = blockIdx.x / cluster;
    const int vocab = p.vocab;
    const TIn* z = static_cast<const TIn*>(p.logits) + row * p.ldLogits;
    // whole vectors start on 16-byte boundaries whatever the row's first address: `shift` elements before it
    const int shift = static_cast<int>((reinterpret_cast<uintptr_t>(z) / sizeof(TIn)) % kN);
    const int vectors = (vocab + shift + kN - 1) / kN;
    const int stride = cluster * blockDim.x;
    const int v0 = rank * blockDim.x + tid;
    const float invTau = 1.0f / p.tau;
    const float c = invTau * kLog2e;

    if (cluster > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");

    uint4 raw[kVecs];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        const int v = v0 + i * stride;
        raw[i] = v < vectors ? distillLoad(z, v * kN - shift, vocab) : make_uint4(0xFF800000u, 0xFF800000u, 0xFF800000u, 0xFF800000u);
        if constexpr (sizeof(TIn) == 2) {
            if (v >= vectors) raw[i] = make_uint4(0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u);
        }
    }
    // the teacher's entries, and the student's logits there, before anything of the row is overwritten
    for (int k = tid; k < p.k; k += blockDim.x) {
        const float idf = p.ids[row * p.k + k];
        const bool finite = fabsf(idf) < 2147483648.0f;
        const int64_t id = finite ? static_cast<int64_t>(lroundf(idf)) : -1;
        const bool ok = id >= 0 && id < vocab;
        sId[k] = ok ? static_cast<int>(id) : -1;
        sQ[k] = !ok ? -INFINITY
                    : p.teacherBf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.teacher)[row * p.k + k])
                                    : static_cast<const float*>(p.teacher)[row * p.k + k];
        sZ[k] = ok ? distillToFloat(z[id]) : 0.0f;
        if (rank == 0 && p.oobCount != nullptr && (!finite || id >= vocab)) atomicAdd(p.oobCount, 1);
    }

    // ---- this warp's maximum and sum of exponentials
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        float v[kN];
        distillUnpack(raw[i], v);
#pragma unroll
        for (int j = 0; j < kN; ++j) top = fmaxf(top, v[j]);
    }
    for (int i = v0 + kVecs * stride; i < vectors; i += stride) {   // beyond the cluster's registers
        float v[kN];
        distillUnpack(distillLoad(z, i * kN - shift, vocab), v);
#pragma unroll
        for (int j = 0; j < kN; ++j) top = fmaxf(top, v[j]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    const float at = top == -INFINITY ? 0.0f : top;   // only -inf so far: exp(-inf - -inf) must not arise
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        float v[kN];
        distillUnpack(raw[i], v);
#pragma unroll
        for (int j = 0; j < kN; ++j) {
            v[j] = exp2f((v[j] - at) * c);
            sum += v[j];
        }
        // fp32: the exponentials take the logits' registers, so that each is computed once
        if constexpr (sizeof(TIn) == 4)
            raw[i] = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
    for (int i = v0 + kVecs * stride; i < vectors; i += stride) {
        float v[kN];
        distillUnpack(distillLoad(z, i * kN - shift, vocab), v);
#pragma unroll
        for (int j = 0; j < kN; ++j) sum += exp2f((v[j] - at) * c);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);

    // ---- exchange over the cluster: one push and one barrier
    const int slot = rank * 32 + warp;
    if (cluster > 1) {
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");   // every block of the cluster runs: its memory may be written
        if (lane < cluster) {
            const uint32_t dst = mapa_cluster(smem_u32(&stats[slot]), static_cast<uint32_t>(lane));
            st_shared_cluster_u32(dst, __float_as_uint(top));
            st_shared_cluster_u32(dst + 4, __float_as_uint(sum));
        }
        cluster_sync_all();
    } else {
        if (lane == 0) stats[slot] = make_float2(top, sum);
        __syncthreads();
    }
    float rowTop = -INFINITY;
    for (int i = lane; i < cluster * 32; i += 32)
        if ((i & 31) < warps) rowTop = fmaxf(rowTop, stats[i].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) rowTop = fmaxf(rowTop, __shfl_xor_sync(0xFFFFFFFFu, rowTop, o));
    const float rowAt = rowTop == -INFINITY ? 0.0f : rowTop;
    float rowSum = 0.0f;
    for (int i = lane; i < cluster * 32; i += 32) {
        if ((i & 31) < warps) {
            const float2 s = stats[i];
            rowSum += s.x == -INFINITY ? s.y : s.y * exp2f((s.x - rowAt) * c);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) rowSum += __shfl_xor_sync(0xFFFFFFFFu, rowSum, o);
    const float logSum = logf(rowSum);

    // ---- the teacher's distribution (first warp), loss and row statistics (first block)
    if (warp == 0) {
        float most = -INFINITY;
        for (int k = lane; k < p.k; k += 32) most = fmaxf(most, sQ[k]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, o));
        float total = 0.0f;
        for (int k = lane; k < p.k; k += 32) {
            if (sId[k] >= 0 && sQ[k] != -INFINITY) total += exp2f((sQ[k] - most) * c);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xFFFFFFFFu, total, o);
        const bool counted = total != 0.0f;   // no entry with any weight: the row does not count
        const float logTotal = logf(total);
        float loss = 0.0f;
        for (int k = lane; k < p.k; k += 32) {
            float q = 0.0f;
            if (sId[k] >= 0 && sQ[k] != -INFINITY) {
                const float logQ = (sQ[k] - most) * invTau - logTotal;
                q = exp2f((sQ[k] - most) * c) / total;
                // q may have underflowed to zero: q log q is zero then, whatever the student holds
                if (q != 0.0f) loss += q * (logQ - ((sZ[k] - rowAt) * invTau - logSum));
            }
            sQ[k] = q;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) loss += __shfl_xor_sync(0xFFFFFFFFu, loss, o);
        if (lane == 0) {
            teacherSum[0] = total;
            if (rank == 0) {
                if (p.loss != nullptr) p.loss[row] = counted ? p.tau * p.tau * loss : 0.0f;
                if (p.lse != nullptr) p.lse[row] = rowTop * invTau + logSum;
            }
        }
    }
    if (p.grad == nullptr) return;
    __syncthreads();
    float g = teacherSum[0] != 0.0f ? ceRowGrad(p.gradLoss, row, p.dGradScale, p.gradScale) * p.tau : 0.0f;

    // ---- gradient of the dense part: p, scaled
    TOut* out = static_cast<TOut*>(p.grad) + row * p.ldGrad;
    const bool aligned = (reinterpret_cast<uintptr_t>(out) - static_cast<uintptr_t>(shift) * sizeof(TOut)) % (kN * sizeof(TOut) < 16 ? 8 : 16) == 0;
    const float warpFactor = (top == -INFINITY ? 0.0f : exp2f((top - rowAt) * c)) / rowSum * g;
    const float rowFactor = g / rowSum;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        const int vi = v0 + i * stride;
        if (vi >= vectors) continue;
        float v[kN];
        distillUnpack(raw[i], v);
#pragma unroll
        for (int j = 0; j < kN; ++j) {
            if constexpr (sizeof(TIn) == 4) v[j] = g != 0.0f ? v[j] * warpFactor : 0.0f;
            else v[j] = g != 0.0f ? exp2f((v[j] - rowAt) * c) * rowFactor : 0.0f;
        }
        distillStore<TOut, kN>(out, vi * kN - shift, vocab, v, aligned);
    }
    for (int vi = v0 + kVecs * stride; vi < vectors; vi += stride) {
        float v[kN];
        distillUnpack(distillLoad(z, vi * kN - shift, vocab), v);
#pragma unroll
        for (int j = 0; j < kN; ++j) v[j] = g != 0.0f ? exp2f((v[j] - rowAt) * c) * rowFactor : 0.0f;
        distillStore<TOut, kN>(out, vi * kN - shift, vocab, v, aligned);
    }
    if (g == 0.0f) return;
    __syncthreads();

    // ---- the teacher's entries: the block that wrote a column corrects it, the first entry for all that name it
    for (int k = tid; k < p.k; k += blockDim.x) {
        const int id = sId[k];
        if (id < 0 || (((id + shift) / kN) / static_cast<int>(blockDim.x)) % cluster != rank) continue;
        bool first = true;
        for (int j = 0; j < k; ++j) first = first && sId[j] != id;
        if (!first) continue;
        float q = sQ[k];
        for (int j = k + 1; j < p.k; ++j) q += sId[j] == id ? sQ[j] : 0.0f;
        const float v = g * (exp2f((sZ[k] - rowAt) * c) / rowSum - q);
        if constexpr (sizeof(TOut) == 4) out[id] = v;
        else out[id] = __float2bfloat16_rn(v);
    }
}

template <typename TIn, typename TOut, int kVecs, int kMaxThreads>
void launchDistill(const DistillParams& p, int64_t rows, int cluster, int threads, cudaStream_t stream) {
    auto kernel = distillKernel<TIn, TOut, kVecs, kMaxThreads>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(rows * cluster));
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = static_cast<size_t>(p.k) * 12;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    BFB_CUDA(cudaLaunchKernelEx(&cfg, kernel, p, cluster));
    noteLaunch();
}

template <typename TIn, typename TOut>
void distillPick(const DistillParams& p, int64_t rows, cudaStream_t stream) {
    constexpr int kN = RowVec<TIn>::kN;
    const int64_t vectors = (p.vocab + 2 * kN - 2) / kN;   // with the largest shift
    auto blocksFor = [&](int threads, int vecs) { return static_cast<int>((vectors + static_cast<int64_t>(threads) * vecs - 1) / (static_cast<int64_t>(threads) * vecs)); };
    if (vectors <= 256) {   // short rows: one block of just the threads it takes
        const int threads = static_cast<int>((vectors + 31) / 32 * 32);
        launchDistill<TIn, TOut, 1, 256>(p, rows, 1, threads, stream);
    } else if (vectors <= 1024) {
        launchDistill<TIn, TOut, 4, 256>(p, rows, 1, 256, stream);
    } else if (blocksFor(256, 8) <= kMaxCluster) {
        launchDistill<TIn, TOut, 8, 256>(p, rows, blocksFor(256, 8), 256, stream);
    } else {
        launchDistill<TIn, TOut, 8, 1024>(p, rows, std::min(kMaxCluster, blocksFor(1024, 8)), 1024, stream);
    }
}

}  // namespace

void distillTopk(const DistillArgs& a, cudaStream_t stream) {
    require(a.dtype == BFB_F32 || a.dtype == BFB_BF16, "distill_topk: logits must be f32 or bf16");
    require(a.teacherDtype == BFB_F32 || a.teacherDtype == BFB_BF16, "distill_topk: teacher logits must be f32 or bf16");
    require(a.grad == nullptr || a.gradDtype == BFB_F32 || a.gradDtype == BFB_BF16, "distill_topk: the gradient must be f32 or bf16");
    require(a.rows >= 0 && a.vocab > 0 && a.k > 0, "distill_topk: sizes must be positive");
    require(a.vocab <= (1ll << 24) && a.rows <= (1ll << 27), "distill_topk: sizes beyond the limits (2^27 rows, 2^24 classes)");
    require(a.k <= kMaxTeacher, "distill_topk: more than 1024 teacher entries a row");
    require(a.tau > 0.0f && a.tau < INFINITY, "distill_topk: the temperature must be positive and finite");
    require(a.ldLogits >= a.vocab && (a.grad == nullptr || a.ldGrad >= a.vocab), "distill_topk: row pitch smaller than vocab");
    if (a.rows == 0) return;
    require(a.logits != nullptr && a.ids != nullptr && a.teacher != nullptr, "distill_topk: null pointer");
    require(a.grad != a.logits || (a.gradDtype == a.dtype && a.ldGrad == a.ldLogits),
            "distill_topk: a gradient in the logits' place has their format and pitch");
    DistillParams p{};
    p.logits = a.logits;
    p.ldLogits = a.ldLogits;
    p.ids = a.ids;
    p.teacher = a.teacher;
    p.teacherBf16 = a.teacherDtype == BFB_BF16;
    p.k = static_cast<int>(a.k);
    p.tau = a.tau;
    p.gradLoss = a.gradLoss;
    p.dGradScale = a.dGradScale;
    p.gradScale = a.gradScale;
    p.loss = a.loss;
    p.lse = a.lse;
    p.grad = a.grad;
    p.ldGrad = a.ldGrad;
    p.vocab = static_cast<int>(a.vocab);
    p.oobCount = a.oobCount;
    const bool outF32 = a.grad != nullptr && a.gradDtype == BFB_F32;
    if (a.dtype == BFB_F32) {
        if (outF32) distillPick<float, float>(p, a.rows, stream);
        else distillPick<float, __nv_bfloat16>(p, a.rows, stream);
    } else {
        if (outF32) distillPick<__nv_bfloat16, float>(p, a.rows, stream);
        else distillPick<__nv_bfloat16, __nv_bfloat16>(p, a.rows, stream);
    }
}

}  // namespace bfb
