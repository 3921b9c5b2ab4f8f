// Distillation from the top logits of a teacher: loss and gradient in one pass over the student's logits.
//
//   q = softmax(teacher / tau) over the listed entries,   p = softmax(z / tau) over the vocabulary
//   loss_t = tau^2 sum_k q_k (log q_k - log p_{i_k}),     dz_tj = g_t tau (p_tj - sum_{k: i_k = j} q_k)
//
// Bound by memory: the least a step can move is the logits once in and the gradient once out. So a row stays on the chip
// between the softmax statistics and the gradient: a cluster of up to eight blocks holds it in shared memory, a slice each that
// arrives as one bulk copy. Every warp pushes its (maximum, sum) into the shared memory of all blocks of the cluster, and
// after one cluster barrier each warp joins all pairs in the same order and finishes its part of the slice. One more warp
// looks after the teacher all the while: entries and their logits while the slice arrives, probabilities, loss and the values
// of the listed columns while the others store the dense gradient. Slices are small enough that several blocks share an
// SM and cover each other's waits; only what a row has beyond the cluster's memory is read again.
// Measured: 8192 x 32000 fp32, k = 64, 431 us = 4.9 TB/s of the 6.56 TB/s a copy reaches; 2047 x 128001 bf16, k = 20, 246 us =
// 4.3 TB/s. What is left is each row's chain (copy, statistics, cluster barrier, join), which five blocks an SM do not cover
// whole. Walking over the rows with two buffers or a ring of chunks and an mbarrier exchange was slower (451 - 730 us): a block
// then waits for its own copies and statistics where other blocks would run.
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
constexpr int kMaxWarps = 16;            // that work on a row's vectors; one more for the teacher
// 42 KiB a block as long as a cluster can hold the row so: five blocks an SM. Measured on 8192 x 32000 fp32 / 2047 x 128001
// bf16 logits (loss and gradient): 22 KiB 491 / 268 us, 32 KiB 445 / 266, 42 KiB 431 / 246, 64 KiB 420 / 268.
constexpr int kSliceVectors = 2688;
constexpr int kMostVectors = 13 * 1024; // 208 KiB: with the entries and statistics within the 227 KiB of a block

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
__device__ __forceinline__ float distillMax(const uint4& raw, float) {
    return fmaxf(fmaxf(__uint_as_float(raw.x), __uint_as_float(raw.y)), fmaxf(__uint_as_float(raw.z), __uint_as_float(raw.w)));
}
__device__ __forceinline__ float distillMax(const uint4& raw, __nv_bfloat16) {
    auto h = [](uint32_t w) { __nv_bfloat162 r; __builtin_memcpy(&r, &w, 4); return r; };
    const __nv_bfloat162 m = __hmax2(__hmax2(h(raw.x), h(raw.y)), __hmax2(h(raw.z), h(raw.w)));
    return fmaxf(__low2float(m), __high2float(m));
}
// 2^x, results below 2^-126 as zero: a probability that small adds nothing to any sum here.
__device__ __forceinline__ float exp2Ftz(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Elements [first, first + kN) of a row of `count`; what lies outside reads as -inf.
template <typename T>
__device__ __forceinline__ uint4 distillEdge(const T* row, int first, int count) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 4) {
            const int at = first + j;
            w[j] = __float_as_uint(at >= 0 && at < count ? row[at] : -INFINITY);
        } else {
            const int at = first + 2 * j;
            const uint32_t lo = at >= 0 && at < count ? __bfloat16_as_ushort(row[at]) : 0xFF80u;
            const uint32_t hi = at + 1 >= 0 && at + 1 < count ? __bfloat16_as_ushort(row[at + 1]) : 0xFF80u;
            w[j] = lo | (hi << 16);
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// The same; whole vectors are 16-byte aligned.
template <typename T>
__device__ __forceinline__ uint4 distillLoad(const T* row, int first, int count) {
    if (first >= 0 && first + RowVec<T>::kN <= count) return *reinterpret_cast<const uint4*>(row + first);
    return distillEdge(row, first, count);
}
// Bulk copy global -> shared of a multiple of 16 bytes between 16-byte boundaries, booked on an mbarrier.
__device__ __forceinline__ void copyBulk(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src),
                 "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}
// kN gradient values as one access (two for 32 bytes).
template <typename T, int kN>
__device__ __forceinline__ void distillStoreVec(T* to, const float (&v)[kN]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < kN; j += 4) __stcs(reinterpret_cast<float4*>(to + j), make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]));
    } else {
        uint32_t w[kN / 2];
#pragma unroll
        for (int j = 0; j < kN / 2; ++j) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);   // the result's format: one rounding
            w[j] = *reinterpret_cast<const uint32_t*>(&h);
        }
        if constexpr (kN == 8) __stcs(reinterpret_cast<uint4*>(to), make_uint4(w[0], w[1], w[2], w[3]));
        else __stcs(reinterpret_cast<uint2*>(to), make_uint2(w[0], w[1]));
    }
}
// The same at `first` of a row; `aligned`: the row's whole vectors can be stored as such.
template <typename T, int kN>
__device__ __forceinline__ void distillStore(T* row, int first, int count, const float (&v)[kN], bool aligned) {
    if (aligned && first >= 0 && first + kN <= count) {
        distillStoreVec<T, kN>(row + first, v);
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

// exp((z - at) c) for many z and one reference: a single multiply-add per value, 2^(z c - high), where high is at * c rounded;
// what the rounding left goes into the factor `rest` of the whole sum. Only where at * c is out of reach (masks of the lowest
// finite value, and nothing else in the batch) is the difference taken first.
struct DistillReference {
    float at, c, high, rest;
    __device__ __forceinline__ DistillReference(float top, float factor) : at(top == -INFINITY ? 0.0f : top), c(factor) {
        high = at * c;
        rest = 1.0f - fmaf(at, c, -high) * kLn2;
        if (!(fabsf(high) < 1e30f)) rest = 1.0f;
    }
    __device__ __forceinline__ bool plain() const { return fabsf(high) < 1e30f; }
    __device__ __forceinline__ float fast(float z) const { return exp2Ftz(fmaf(z, c, -high)); }
    __device__ __forceinline__ float slow(float z) const { return exp2Ftz((z - at) * c); }
};

// (maximum, sum of exp((z - maximum) c)) of a thread brought forward by kBatch vectors. While nothing but -inf has been seen
// the reference point is 0, so that exp(-inf - -inf) never arises; a NaN reaches the sum and stays there.
template <typename T, int kBatch>
__device__ __forceinline__ void distillAccumulate(const uint4 (&raw)[kBatch], float c, float& top, float& sum) {
    constexpr int kN = RowVec<T>::kN;
    float most = distillMax(raw[0], T{});
#pragma unroll
    for (int u = 1; u < kBatch; ++u) most = fmaxf(most, distillMax(raw[u], T{}));
    if (most > top) {
        sum = top == -INFINITY ? sum : sum * exp2Ftz((top - most) * c);
        top = most;
    }
    const DistillReference ref(top, c);
    float part[2] = {0.0f, 0.0f};
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
        float v[kN];
        distillUnpack(raw[u], v);
        if (ref.plain()) {
#pragma unroll
            for (int j = 0; j < kN; ++j) part[j & 1] += ref.fast(v[j]);
        } else {
#pragma unroll
            for (int j = 0; j < kN; ++j) part[j & 1] += ref.slow(v[j]);
        }
    }
    sum += (part[0] + part[1]) * ref.rest;
}

// `held`: vectors of the row a block keeps in shared memory; what the row has beyond cluster * held of them is read from
// global memory in both passes.
template <typename TIn, typename TOut>
__global__ void __launch_bounds__(kMaxWarps * 32 + 32, 2)
distillKernel(const DistillParams p, int cluster, int held) {
    constexpr int kN = RowVec<TIn>::kN;
    __shared__ alignas(8) uint64_t fullBar;              // the slice has arrived
    __shared__ float2 stats[kMaxCluster * kMaxWarps];   // (maximum, sum) of every warp of the cluster, block by block
    __shared__ int counted;                              // some entry has weight: the row counts
    __shared__ int abortWord;
    extern __shared__ uint4 dyn[];
    uint4* slice = dyn;                                  // [held]
    const int kPad = (p.k + 3) & ~3;
    int* sId = reinterpret_cast<int*>(dyn + held);       // [k, padded]: column, -1 for an entry left out
    float* sQ = reinterpret_cast<float*>(sId + kPad);    // teacher's logit, then probability
    float* sZ = sQ + kPad;                               // the student's logit, then the gradient of the column

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int threads = blockDim.x - 32, warps = threads >> 5;   // those that work on the row's vectors
    const int rank = static_cast<int>(cluster_ctarank());
    const int64_t row = blockIdx.x / cluster;
    const int vocab = p.vocab;
    const TIn* z = static_cast<const TIn*>(p.logits) + row * p.ldLogits;
    // whole vectors start on 16-byte boundaries whatever the row's first address: `shift` elements before it
    const int shift = static_cast<int>((reinterpret_cast<uintptr_t>(z) / sizeof(TIn)) % kN);
    const int vectors = (vocab + shift + kN - 1) / kN;
    const int v0 = rank * held;                          // first vector held here
    const int mine = max(0, min(held, vectors - v0));
    const int beyond = cluster * held;                   // vectors from here on are nobody's: taken in turn
    // vectors in [from, to) of the slice lie in the row as a whole
    const int from = v0 == 0 && shift > 0 ? 1 : 0;
    const int to = min(mine, (vocab + shift) / kN - v0);
    const float invTau = 1.0f / p.tau;
    const float c = invTau * kLog2e;

    if (cluster > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");

    float top = -INFINITY, sum = 0.0f;
    if (warp == warps) {
        // ---- the teacher's entries and the student's logits there, before anything of the row is overwritten
        bool any = false;
        for (int k0 = lane; k0 < kPad; k0 += 128) {   // four entries a lane at a time: two trips to memory, not eight
            float idf[4], t[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int k = k0 + 32 * u;
                idf[u] = k < p.k ? p.ids[row * p.k + k] : -1.0f;
                t[u] = k >= p.k ? -INFINITY
                                : p.teacherBf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.teacher)[row * p.k + k])
                                                : static_cast<const float*>(p.teacher)[row * p.k + k];
            }
            int id[4];
            float zk[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const bool finite = fabsf(idf[u]) < 2147483648.0f;
                const int64_t wide = finite ? static_cast<int64_t>(lroundf(idf[u])) : -1;
                if (rank == 0 && p.oobCount != nullptr && (!finite || wide >= vocab)) atomicAdd(p.oobCount, 1);
                id[u] = wide >= 0 && wide < vocab && t[u] != -INFINITY ? static_cast<int>(wide) : -1;
                zk[u] = id[u] >= 0 ? distillToFloat(z[id[u]]) : 0.0f;
                any = any || id[u] >= 0;
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int k = k0 + 32 * u;
                if (k >= kPad) break;
                sId[k] = id[u];
                sQ[k] = t[u];
                sZ[k] = zk[u];
            }
        }
        any = __any_sync(0xFFFFFFFFu, any);
        if (lane == 0) counted = any;
    } else {
        // ---- the slice, then this warp's maximum and sum of exponentials
        if (tid == 0) {
            abortWord = 0;
            mbar_init(&fullBar, 1);
            fence_mbar_init();
            if (to > from) {
                mbar_arrive_expect_tx(&fullBar, static_cast<uint32_t>(to - from) * 16);
                copyBulk(slice + from, z + ((v0 + from) * kN - shift), static_cast<uint32_t>(to - from) * 16, &fullBar);
            } else {
                mbar_arrive(&fullBar);
            }
            if (from > 0) slice[0] = distillEdge(z, -shift, vocab);
        }
        if (tid == (warps > 1 ? 32 : 1) && to < mine && mine - 1 >= from) slice[mine - 1] = distillEdge(z, (v0 + mine - 1) * kN - shift, vocab);
        asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory");
        mbar_wait(&fullBar, 0, &abortWord, nullptr, kDevTimeoutOther);
        int i = tid;
        for (; i + 3 * threads < mine; i += 4 * threads) {
            const uint4 raw[4] = {slice[i], slice[i + threads], slice[i + 2 * threads], slice[i + 3 * threads]};
            distillAccumulate<TIn, 4>(raw, c, top, sum);
        }
        for (; i < mine; i += threads) {
            const uint4 raw[1] = {slice[i]};
            distillAccumulate<TIn, 1>(raw, c, top, sum);
        }
        for (int vi = beyond + rank * threads + tid; vi < vectors; vi += cluster * threads) {
            const uint4 raw[1] = {distillLoad(z, vi * kN - shift, vocab)};
            distillAccumulate<TIn, 1>(raw, c, top, sum);
        }
        float most = top;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, o));
        sum = top == -INFINITY ? sum : sum * exp2Ftz((top - most) * c);
        top = most;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        if (abortWord != 0) sum = NAN;   // the copy never came: nothing that follows is a number
    }

    // ---- exchange over the cluster: one push and one barrier
    const int slot = rank * kMaxWarps + warp;
    if (cluster > 1) {
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");   // every block of the cluster runs: its memory may be written
        if (warp < warps && lane < cluster) {
            const uint32_t dst = mapa_cluster(smem_u32(&stats[slot]), static_cast<uint32_t>(lane));
            st_shared_cluster_u32(dst, __float_as_uint(top));
            st_shared_cluster_u32(dst + 4, __float_as_uint(sum));
        }
        cluster_sync_all();
    } else {
        if (warp < warps && lane == 0) stats[slot] = make_float2(top, sum);
        __syncthreads();
    }
    float2 part[kMaxCluster * kMaxWarps / 32];
    float rowTop = -INFINITY;
#pragma unroll
    for (int s = 0; s < kMaxCluster * kMaxWarps / 32; ++s) {
        const int at = s * 32 + lane;
        part[s] = at < cluster * kMaxWarps && at % kMaxWarps < warps ? stats[at] : make_float2(-INFINITY, 0.0f);
        rowTop = fmaxf(rowTop, part[s].x);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) rowTop = fmaxf(rowTop, __shfl_xor_sync(0xFFFFFFFFu, rowTop, o));
    const float rowAt = rowTop == -INFINITY ? 0.0f : rowTop;
    float rowSum = 0.0f;
#pragma unroll
    for (int s = 0; s < kMaxCluster * kMaxWarps / 32; ++s) {
        if (s * 32 < cluster * kMaxWarps) rowSum += part[s].x == -INFINITY ? part[s].y : part[s].y * exp2Ftz((part[s].x - rowAt) * c);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) rowSum += __shfl_xor_sync(0xFFFFFFFFu, rowSum, o);
    const float g = counted != 0 && p.grad != nullptr ? ceRowGrad(p.gradLoss, row, p.dGradScale, p.gradScale) * p.tau : 0.0f;
    TOut* out = static_cast<TOut*>(p.grad) + (p.grad != nullptr ? row * p.ldGrad : 0);

    if (warp == warps) {
        // ---- the teacher's distribution, loss and row statistics, and the gradient of the columns that are listed
        float most = -INFINITY;
        for (int k = lane; k < p.k; k += 32)
            if (sId[k] >= 0) most = fmaxf(most, sQ[k]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, o));
        float total = 0.0f;
        for (int k = lane; k < p.k; k += 32)
            if (sId[k] >= 0) total += exp2Ftz((sQ[k] - most) * c);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xFFFFFFFFu, total, o);
        const float logSum = logf(rowSum), logTotal = logf(total), inverse = 1.0f / total;
        float loss = 0.0f;
        for (int k = lane; k < kPad; k += 32) {
            float q = 0.0f;
            if (sId[k] >= 0) {
                const float t = sQ[k] - most;
                q = exp2Ftz(t * c) * inverse;
                // q may have underflowed to zero: q log q is zero then, whatever the student holds
                if (q != 0.0f) loss += q * (t * invTau - logTotal - ((sZ[k] - rowAt) * invTau - logSum));
            }
            sQ[k] = q;
        }
        if (rank == 0) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) loss += __shfl_xor_sync(0xFFFFFFFFu, loss, o);
            if (lane == 0) {
                if (p.loss != nullptr) p.loss[row] = counted != 0 ? p.tau * p.tau * loss : 0.0f;
                if (p.lse != nullptr) p.lse[row] = rowTop * invTau + logSum;
            }
        }
        if (g == 0.0f) return;   // no gradient, or zero everywhere (nobody waits then, see below)
        __syncwarp();
        for (int k = lane; k < p.k; k += 32) {
            const int id = sId[k];
            if (id < 0) continue;
            // the block that stores a column corrects it; all entries that name it count
            const int vi = (id + shift) / kN;
            if ((vi < beyond ? vi / held : (vi - beyond) / threads % cluster) != rank) continue;
            float q = 0.0f;
            for (int j = 0; j < kPad; j += 4) {
                const int4 other = *reinterpret_cast<const int4*>(sId + j);
                const float4 weight = *reinterpret_cast<const float4*>(sQ + j);
                q += (other.x == id ? weight.x : 0.0f) + (other.y == id ? weight.y : 0.0f) + (other.z == id ? weight.z : 0.0f) +
                     (other.w == id ? weight.w : 0.0f);
            }
            sZ[k] = g * (exp2Ftz((sZ[k] - rowAt) * c) / rowSum - q);
        }
        __syncthreads();   // the dense gradient is stored
        for (int k = lane; k < p.k; k += 32) {
            const int id = sId[k];
            if (id < 0) continue;
            const int vi = (id + shift) / kN;
            if ((vi < beyond ? vi / held : (vi - beyond) / threads % cluster) != rank) continue;
            // entries that name the same column have the same value
            if constexpr (sizeof(TOut) == 4) out[id] = sZ[k];
            else out[id] = __float2bfloat16_rn(sZ[k]);
        }
        return;
    }
    if (p.grad == nullptr) return;

    // ---- gradient of the dense part: p, scaled
    const bool aligned = (reinterpret_cast<uintptr_t>(out) - static_cast<uintptr_t>(shift) * sizeof(TOut)) % (kN * sizeof(TOut) < 16 ? 8 : 16) == 0;
    const DistillReference ref(rowTop, c);
    const float factor = g / rowSum * ref.rest;
    auto finish = [&](const uint4& raw, float (&v)[kN]) {
        distillUnpack(raw, v);
#pragma unroll
        for (int j = 0; j < kN; ++j) v[j] = g == 0.0f ? 0.0f : (ref.plain() ? ref.fast(v[j]) : ref.slow(v[j])) * factor;   // zero whatever the logits hold
    };
    TOut* const dst = out + (v0 * kN - shift);
    const bool quick = g != 0.0f && ref.plain() && aligned;
    int i = tid;
    if (quick && from <= i) {
        for (; i + threads < to; i += 2 * threads) {
            const uint4 raw[2] = {slice[i], slice[i + threads]};
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float v[kN];
                distillUnpack(raw[u], v);
#pragma unroll
                for (int q = 0; q < kN; ++q) v[q] = ref.fast(v[q]) * factor;
                distillStoreVec<TOut, kN>(dst + (i + u * threads) * kN, v);
            }
        }
    }
    for (; i < mine; i += threads) {
        float v[kN];
        finish(slice[i], v);
        if (aligned && i >= from && i < to) distillStoreVec<TOut, kN>(dst + i * kN, v);
        else distillStore<TOut, kN>(out, (v0 + i) * kN - shift, vocab, v, false);
    }
    for (int vi = beyond + rank * threads + tid; vi < vectors; vi += cluster * threads) {
        float v[kN];
        finish(distillLoad(z, vi * kN - shift, vocab), v);
        distillStore<TOut, kN>(out, vi * kN - shift, vocab, v, aligned);
    }
    if (g != 0.0f) __syncthreads();
}

template <typename TIn, typename TOut>
void launchDistill(const DistillParams& p, int64_t rows, cudaStream_t stream) {
    constexpr int kN = RowVec<TIn>::kN;
    const int64_t vectors = (p.vocab + 2 * kN - 2) / kN;   // with the largest shift
    // as few blocks as hold the row at 42 KiB each, then as much as it takes in eight blocks
    const int cluster = static_cast<int>(std::min<int64_t>(kMaxCluster, (vectors + kSliceVectors - 1) / kSliceVectors));
    const int held = static_cast<int>(std::min<int64_t>((vectors + cluster - 1) / cluster, kMostVectors));
    // sixteen vectors a thread (six: 742 / 396 us instead of 431 / 246, the joins of the statistics are per warp), and a warp
    // for the teacher
    const int threads = static_cast<int>(std::min<int64_t>(kMaxWarps * 32, std::max<int64_t>(32, (held / 16 + 31) / 32 * 32))) + 32;
    auto kernel = distillKernel<TIn, TOut>;
    const size_t smem = static_cast<size_t>(held) * 16 + static_cast<size_t>((p.k + 3) / 4 * 4) * 12;
    BFB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(rows * cluster));
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    BFB_CUDA(cudaLaunchKernelEx(&cfg, kernel, p, cluster, held));
    noteLaunch();
}

}  // namespace

void distillTopk(const DistillArgs& a, cudaStream_t stream) {
    require(a.dtype == BFB_F32 || a.dtype == BFB_BF16, "distill_topk: logits must be f32 or bf16");
    require(a.teacherDtype == BFB_F32 || a.teacherDtype == BFB_BF16, "distill_topk: teacher logits must be f32 or bf16");
    require(a.grad == nullptr || a.gradDtype == BFB_F32 || a.gradDtype == BFB_BF16, "distill_topk: the gradient must be f32 or bf16");
    require(a.rows >= 0 && a.vocab > 0 && a.k > 0, "distill_topk: sizes must be positive");
    require(a.vocab <= (1ll << 24) && a.rows <= (1ll << 27), "distill_topk: sizes beyond the limits (2^27 rows, 2^24 classes)");
    require(a.k <= kMaxTeacher, "distill_topk: more than 1024 teacher entries a row");
    require(a.tau >= 1e-6f && a.tau <= 1e6f, "distill_topk: the temperature must be within 1e-6 .. 1e6");
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
        if (outF32) launchDistill<float, float>(p, a.rows, stream);
        else launchDistill<float, __nv_bfloat16>(p, a.rows, stream);
    } else {
        if (outF32) launchDistill<__nv_bfloat16, float>(p, a.rows, stream);
        else launchDistill<__nv_bfloat16, __nv_bfloat16>(p, a.rows, stream);
    }
}

}  // namespace bfb
