// Embedding lookup with a scale, and the gradient of the table by sorted tokens.
//
//   out_t = scale * E[id_t],      dE_v = scale * sum_{t: id_t = v} dout_t
//
// Both are bound by memory. The gradient reads dout once and writes the table once, with no atomics, so that its bits do not
// depend on timing:
//   1. sortTokensKernel orders the token positions by id (stable: positions of one id stay ascending). One cluster of up
//      to eight blocks does all digits of a radix sort in one launch, its counters joined over distributed shared memory.
//   2. embedReduceKernel cuts the sorted list into pieces of equal length whatever ids they hold, so that a token that makes
//      up a third of the text costs what any other rows cost. A block sums a piece's rows in fp32 and stores each id whose
//      whole run lies inside; the ends of runs that cross a border go to a small array. Other blocks of the same launch
//      write the rows of ids that do not occur.
//   3. embedJoinKernel adds up the parts of the runs that crossed borders, in order.
// Measured with 65536 tokens, 32000 x 2048 fp32, token frequencies that fall with the rank: lookup 117 us, sort 35, reduction 134
// (800 MB, 6.0 TB/s), joins 19; 306 us together = 5.2 TB/s of the 6.56 TB/s a copy reaches. The sort is bound by its two
// passes of ranking 32 pairs at a time in the eight blocks of one cluster.
#include <cuda_bf16.h>

#include <algorithm>
#include <climits>

#include "common.cuh"
#include "kernels.hpp"
#include "ptx_sm100.cuh"

namespace bfb {

namespace {

constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortCluster = 8;
constexpr int kMaxDigitBits = 9;
constexpr int kMaxPiece = 128;      // most sorted entries per block of the reduction
constexpr int kZeroRows = 64;       // table rows a block looks after when it writes the rows that do not occur
constexpr int kReduceThreads = 256;

inline int64_t roundUp(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
inline bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Token ids are float32 holding integers; one outside [0, vocab) names no row (`vocab` comes back). Rounded to the nearest,
// halves away from zero (lroundf) in 32 bits: the conversions to 64 are what the sort's first pass would spend its time on.
__device__ __forceinline__ uint32_t tokenRow(float idf, int64_t vocab) {
    if (!(fabsf(idf) < 16777217.0f)) return static_cast<uint32_t>(vocab);   // beyond every table (2^24 rows), infinite, NaN
    float whole = truncf(idf);
    if (fabsf(idf - whole) >= 0.5f) whole += copysignf(1.0f, idf);
    const int id = __float2int_rz(whole);
    return id >= 0 && id < static_cast<int>(vocab) ? static_cast<uint32_t>(id) : static_cast<uint32_t>(vocab);
}

template <typename T>
__device__ __forceinline__ float toFloat(T v);
template <>
__device__ __forceinline__ float toFloat<float>(float v) { return v; }
template <>
__device__ __forceinline__ float toFloat<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T fromFloat(float v);
template <>
__device__ __forceinline__ float fromFloat<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 fromFloat<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// kN neighbouring elements, aligned to their size up to 16 bytes.
template <typename T, int kN>
struct alignas(sizeof(T) * kN < 16 ? sizeof(T) * kN : 16) Pack {
    T v[kN];
};

// ---- lookup --------------------------------------------------------------------------------------------------

// blockDim.x threads across a row's packs, blockDim.y groups of kTokens tokens: the ids, then the rows of a group are all in
// flight at once.
constexpr int kTokens = 4;

template <typename TIn, typename TOut, int kN>
__global__ void __launch_bounds__(256)
embedScaledKernel(const float* __restrict__ ids, const TIn* __restrict__ table, TOut* __restrict__ out, int64_t ldOut, int64_t tokens,
                  int64_t vocab, int64_t dim, float scale, int* oobCount) {
    const int64_t packs = dim / kN;
    const int64_t groups = (tokens + kTokens - 1) / kTokens;
    for (int64_t group = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y; group < groups; group += static_cast<int64_t>(gridDim.x) * blockDim.y) {
        const int64_t t0 = group * kTokens;
        uint32_t id[kTokens];
#pragma unroll
        for (int u = 0; u < kTokens; ++u) id[u] = t0 + u < tokens ? tokenRow(__ldg(ids + t0 + u), vocab) : static_cast<uint32_t>(vocab);
        if (threadIdx.x == 0 && oobCount != nullptr) {
#pragma unroll
            for (int u = 0; u < kTokens; ++u)
                if (t0 + u < tokens && id[u] >= vocab) atomicAdd(oobCount, 1);
        }
        for (int64_t i = threadIdx.x; i < packs; i += blockDim.x) {
            Pack<TIn, kN> v[kTokens];
#pragma unroll
            for (int u = 0; u < kTokens; ++u)
                if (id[u] < vocab) v[u] = reinterpret_cast<const Pack<TIn, kN>*>(table + static_cast<int64_t>(id[u]) * dim)[i];
#pragma unroll
            for (int u = 0; u < kTokens; ++u) {
                if (t0 + u >= tokens) break;
                Pack<TOut, kN> r;
#pragma unroll
                for (int j = 0; j < kN; ++j) r.v[j] = fromFloat<TOut>(id[u] < vocab ? toFloat(v[u].v[j]) * scale : 0.0f);
                reinterpret_cast<Pack<TOut, kN>*>(out + (t0 + u) * ldOut)[i] = r;
            }
        }
    }
}

// ---- 1. sort -------------------------------------------------------------------------------------------------

// (row, token position) in one word of eight bytes: a place in the sorted list costs one scattered store, and those are what a
// pass of the sort is made of.
struct SortBuffers {
    uint2* pairs[2];
};

// Stable radix sort of (row, position) pairs, `passes` digits of `bits` bits. The cluster's blocks, their warps and a
// warp's batches of 32 take consecutive stretches of the list; a pair's place is: all smaller digits, the same digit in
// stretches before its own, the same digit before it in its batch. Rows that name no id (vocab) end up last. `occurs` gets a
// bit for every row that is named.
__global__ void __launch_bounds__(kSortThreads, 1)
sortTokensKernel(const float* __restrict__ ids, SortBuffers buf, uint32_t* __restrict__ occurs, int64_t count, int64_t vocab, int passes, int bits,
                 int cluster) {
    pdl_launch_dependents();   // the reduction may set itself up; it waits for the sorted lists
    extern __shared__ uint32_t counts[];   // [kSortWarps][bins], then [bins] totals of this block, [bins] bases
    const int bins = 1 << bits;
    uint32_t* blockTotal = counts + kSortWarps * bins;
    uint32_t* base = blockTotal + bins;
    __shared__ uint32_t warpScan[kSortWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = static_cast<int>(cluster_ctarank());
    const int64_t perWarp = (count + static_cast<int64_t>(cluster) * kSortWarps * 32 - 1) / (static_cast<int64_t>(cluster) * kSortWarps * 32) * 32;
    const int64_t begin = min(count, (static_cast<int64_t>(rank) * kSortWarps + warp) * perWarp);
    const int64_t end = min(count, begin + perWarp);
    uint32_t* mine = counts + warp * bins;
    // warps of this block that have a stretch
    const int64_t before0 = static_cast<int64_t>(rank) * kSortWarps * perWarp;
    const int active = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(kSortWarps), (count - before0 + perWarp - 1) / perWarp)));
    const int64_t all32 = static_cast<int64_t>(cluster) * kSortThreads, me = static_cast<int64_t>(rank) * kSortThreads + tid;
    for (int64_t i = me; i < (vocab + 31) / 32; i += all32) occurs[i] = 0;
    constexpr int kBatch = 8;   // loads in flight per lane
    for (int pass = 0; pass < passes; ++pass) {
        const int shift = pass * bits;
        const uint2* src = buf.pairs[(pass & 1) ^ 1];
        uint2* dst = buf.pairs[pass & 1];
        // the stretch's pairs from i0 on, a batch per lane; all loads first, whatever lies behind the end reads the last one again
        auto pairsAt = [&](int64_t i0, uint2 (&pair)[kBatch]) {
            if (pass == 0) {
                float id[kBatch];
#pragma unroll
                for (int u = 0; u < kBatch; ++u) id[u] = __ldg(ids + min(i0 + 32 * u + lane, end - 1));
#pragma unroll
                for (int u = 0; u < kBatch; ++u) pair[u] = make_uint2(tokenRow(id[u], vocab), static_cast<uint32_t>(i0 + 32 * u + lane));
            } else {
#pragma unroll
                for (int u = 0; u < kBatch; ++u) pair[u] = __ldcg(src + min(i0 + 32 * u + lane, end - 1));
            }
        };
        for (int i = tid; i < active * bins; i += kSortThreads) counts[i] = 0;
        __syncthreads();
        uint2 pair[kBatch];   // of a stretch that is one batch, for both its uses
        for (int64_t i0 = begin; i0 < end; i0 += 32 * kBatch) {
            pairsAt(i0, pair);
#pragma unroll
            for (int u = 0; u < kBatch; ++u)
                if (i0 + 32 * u + lane < end) atomicAdd(&mine[(pair[u].x >> shift) & (bins - 1)], 1u);
        }
        __syncthreads();
        // per digit: what the block's earlier warps hold, and the block's total
        if (tid < bins) {
            uint32_t total = 0;
            for (int w0 = 0; w0 < active; w0 += 8) {
                uint32_t held[8];
#pragma unroll
                for (int w = 0; w < 8; ++w) held[w] = w0 + w < active ? counts[(w0 + w) * bins + tid] : 0;
#pragma unroll
                for (int w = 0; w < 8; ++w) {
                    if (w0 + w < active) counts[(w0 + w) * bins + tid] = total;
                    total += held[w];
                }
            }
            blockTotal[tid] = total;
        }
        if (cluster > 1) cluster_sync_all();
        else __syncthreads();
        // per digit: all blocks' totals, and those of the blocks before this one
        uint32_t all = 0, before = 0;
        if (tid < bins) {
            uint32_t theirs[kSortCluster];
#pragma unroll
            for (int r = 0; r < kSortCluster; ++r) {
                theirs[r] = 0;
                if (r < cluster) {
                    const uint32_t from = mapa_cluster(smem_u32(&blockTotal[tid]), static_cast<uint32_t>(r));
                    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(theirs[r]) : "r"(from) : "memory");
                }
            }
#pragma unroll
            for (int r = 0; r < kSortCluster; ++r) {
                all += theirs[r];
                before += r < rank ? theirs[r] : 0;
            }
        }
        uint32_t scan = all;   // inclusive over the digits
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t n = __shfl_up_sync(0xFFFFFFFFu, scan, o);
            if (lane >= o) scan += n;
        }
        if (lane == 31) warpScan[warp] = scan;
        __syncthreads();
        uint32_t smaller = 0;
        for (int w = 0; w < warp; ++w) smaller += warpScan[w];
        if (tid < bins) base[tid] = smaller + scan - all + before;
        __syncthreads();
        // places, 32 pairs at a time
        for (int64_t i0 = begin; i0 < end; i0 += 32 * kBatch) {
            if (end - begin > 32 * kBatch) pairsAt(i0, pair);
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                if (i0 + 32 * u >= end) break;
                const bool live = i0 + 32 * u + lane < end;
                const uint32_t digit = live ? (pair[u].x >> shift) & (bins - 1) : 0xFFFFFFFFu;
                const uint32_t same = __match_any_sync(0xFFFFFFFFu, digit);
                if (live) {
                    const uint32_t earlier = __popc(same & ((1u << lane) - 1u));
                    const uint32_t at = base[digit] + mine[digit] + earlier;
                    if (at < count) dst[at] = pair[u];   // always, unless the ids change while the kernel runs
                }
                __syncwarp();
                if (live && lane == 31 - __clz(same)) mine[digit] += __popc(same);
                __syncwarp();
            }
        }
        // the next pass reads what other blocks wrote; and nobody leaves while its totals are being read
        __threadfence();
        if (cluster > 1) cluster_sync_all();
        else __syncthreads();
    }
    // where a run begins: its row occurs
    const uint2* sorted = buf.pairs[(passes - 1) & 1];
    for (int64_t i0 = me; i0 < count; i0 += all32 * 4) {
        uint32_t key[4], before[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t i = i0 + u * all32;
            key[u] = i < count ? __ldcg(&sorted[i].x) : static_cast<uint32_t>(vocab);
            before[u] = i > 0 && i < count ? __ldcg(&sorted[i - 1].x) : 0xFFFFFFFFu;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (key[u] < vocab && key[u] != before[u]) atomicOr(occurs + (key[u] >> 5), 1u << (key[u] & 31));
    }
}

// ---- 2. sums of the sorted rows ---------------------------------------------------------------------------------

struct ReduceParams {
    const uint2* pairs;        // sorted (row, token position)
    const uint32_t* occurs;    // a bit for every row that is named (null: none is)
    int64_t count;             // entries, those that name no row last
    int64_t vocab, dim;
    const void* dout;
    int64_t ldDout;
    void* dtable;
    float scale;
    int accumulate;
    float* ends;               // [pieces][2][dim]: sums of a piece's first run (begun earlier) and last run (going on)
    int64_t pieces;
    int piece;                 // entries a piece
    int64_t columnBlocks;
};

template <typename T, int kN>
__device__ __forceinline__ void storeRow(T* row, int64_t pack, const float (&acc)[kN], float scale, bool accumulate) {
    auto* dst = reinterpret_cast<Pack<T, kN>*>(row) + pack;
    Pack<T, kN> r;
    if (accumulate) {
        const Pack<T, kN> old = *dst;
#pragma unroll
        for (int j = 0; j < kN; ++j) r.v[j] = fromFloat<T>(fmaf(acc[j], scale, toFloat(old.v[j])));
    } else {
#pragma unroll
        for (int j = 0; j < kN; ++j) r.v[j] = fromFloat<T>(acc[j] * scale);
    }
    *dst = r;
}

template <typename TIn, typename TOut, int kN>
__global__ void __launch_bounds__(kReduceThreads)
embedReduceKernel(const ReduceParams p) {
    pdl_launch_dependents();
    pdl_wait();
    __shared__ uint32_t sKey[kMaxPiece + 2], sValue[kMaxPiece];
    const int64_t reduceBlocks = p.pieces * p.columnBlocks;
    const int tid = threadIdx.x;
    if (blockIdx.x < reduceBlocks) {
        const int64_t piece = blockIdx.x / p.columnBlocks;
        const int64_t pack = (blockIdx.x % p.columnBlocks) * kReduceThreads + tid;
        const int64_t begin = piece * p.piece;
        const int n = static_cast<int>(min(static_cast<int64_t>(p.piece), p.count - begin));
        // the piece with its neighbours on both sides; `vocab` stands for no row
        const uint32_t none = static_cast<uint32_t>(p.vocab);
        if (tid < n + 2) {
            const int64_t i = begin + tid - 1;
            const uint2 pair = i >= 0 && i < p.count ? p.pairs[i] : make_uint2(none, 0);
            sKey[tid] = pair.x;
            if (tid >= 1 && tid <= n) sValue[tid - 1] = pair.y;
        }
        __syncthreads();
        if (pack * kN >= p.dim) return;
        const TIn* dout = static_cast<const TIn*>(p.dout) + pack * kN;
        TOut* table = static_cast<TOut*>(p.dtable);
        float acc[kN] = {};
        int runBegin = 0;
        auto flush = [&](int runEnd) {   // entries [runBegin, runEnd) of the piece are one run
            const uint32_t key = sKey[runBegin + 1];
            const bool begun = runBegin == 0 && sKey[0] == key;
            const bool goesOn = runEnd == n && sKey[n + 1] == key;
            if (begun || goesOn) {
                float* end = p.ends + (piece * 2 + (begun ? 0 : 1)) * p.dim + pack * kN;
#pragma unroll
                for (int j = 0; j < kN; ++j) end[j] = acc[j];
            } else {
                storeRow<TOut, kN>(table + static_cast<int64_t>(key) * p.dim, pack, acc, p.scale, p.accumulate != 0);
            }
        };
        constexpr int kAhead = 8;
        for (int i0 = 0; i0 < n; i0 += kAhead) {
            Pack<TIn, kN> v[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                if (i0 + u < n && sKey[i0 + u + 1] != none)
                    v[u] = *reinterpret_cast<const Pack<TIn, kN>*>(dout + static_cast<int64_t>(sValue[i0 + u]) * p.ldDout);
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int i = i0 + u;
                if (i >= n || sKey[i + 1] == none) break;
                if (i > runBegin && sKey[i + 1] != sKey[i]) {
                    flush(i);
                    runBegin = i;
#pragma unroll
                    for (int j = 0; j < kN; ++j) acc[j] = 0.0f;
                }
#pragma unroll
                for (int j = 0; j < kN; ++j) acc[j] += toFloat(v[u].v[j]);
            }
        }
        // the last run ends with the piece or where the entries without a row begin
        int live = n;
        while (live > 0 && sKey[live] == none) --live;
        if (live > 0) {
            if (live == n) {
                flush(n);
            } else {
                const uint32_t key = sKey[runBegin + 1];
                if (runBegin == 0 && sKey[0] == key) {
                    float* end = p.ends + piece * 2 * p.dim + pack * kN;
#pragma unroll
                    for (int j = 0; j < kN; ++j) end[j] = acc[j];
                } else {
                    storeRow<TOut, kN>(table + static_cast<int64_t>(key) * p.dim, pack, acc, p.scale, p.accumulate != 0);
                }
            }
        }
        return;
    }
    // ---- rows that do not occur: a block looks after kZeroRows neighbouring rows
    const int64_t row0 = (blockIdx.x - reduceBlocks) * kZeroRows;
    const int rows = static_cast<int>(min(static_cast<int64_t>(kZeroRows), p.vocab - row0));
    uint32_t seen[kZeroRows / 32];
#pragma unroll
    for (int w = 0; w < kZeroRows / 32; ++w) seen[w] = p.occurs != nullptr && row0 + w * 32 < p.vocab ? p.occurs[row0 / 32 + w] : 0;
    auto occurs = [&](int r) { return ((r < 32 ? seen[0] : seen[1]) >> (r & 31)) & 1u; };
    static_assert(kZeroRows == 64, "two words of the map per block");
    TOut* table = static_cast<TOut*>(p.dtable);
    int r = 0;
    while (r < rows) {
        if (occurs(r)) {
            ++r;
            continue;
        }
        int to = r + 1;   // a stretch of rows without a token is one stretch of memory
        while (to < rows && !occurs(to)) ++to;
        char* from = reinterpret_cast<char*>(table + (row0 + r) * p.dim);
        const int64_t bytes = static_cast<int64_t>(to - r) * p.dim * static_cast<int64_t>(sizeof(TOut));
        const int64_t head = min(bytes, static_cast<int64_t>((16 - reinterpret_cast<uintptr_t>(from) % 16) % 16));
        const int64_t body = (bytes - head) / 16;
        for (int64_t i = tid; i < head / static_cast<int64_t>(sizeof(TOut)); i += blockDim.x) reinterpret_cast<TOut*>(from)[i] = fromFloat<TOut>(0.0f);
        for (int64_t i = tid; i < body; i += blockDim.x) __stcs(reinterpret_cast<uint4*>(from + head) + i, make_uint4(0, 0, 0, 0));
        for (int64_t i = head + body * 16 + tid * static_cast<int64_t>(sizeof(TOut)); i < bytes; i += blockDim.x * static_cast<int64_t>(sizeof(TOut)))
            *reinterpret_cast<TOut*>(from + i) = fromFloat<TOut>(0.0f);
        r = to;
    }
}

// ---- 3. runs that cross the borders of pieces --------------------------------------------------------------------

// A piece whose last run goes on, and did not begin before the piece, starts a chain: its own part, then the first parts of
// the pieces behind it that begin with the same row. Most blocks find no chain, or one that ends with the next piece, so a
// block takes as many columns as its threads hold (kN each). Where a row is narrower than that, the threads left over form
// groups that share a long chain batch by batch; their sums are joined in order.
template <typename TOut, int kN>
__global__ void __launch_bounds__(256)
embedJoinKernel(const ReduceParams p, int groupThreads) {
    __shared__ float joined[256 * kN];
    pdl_wait();
    const int64_t piece = blockIdx.x;
    const int64_t begin = piece * p.piece, next = begin + p.piece;   // piece + 1 < pieces: `next` is an entry
    const uint32_t key = p.pairs[next - 1].x, following = p.pairs[next].x, first = p.pairs[begin].x, earlier = begin > 0 ? p.pairs[begin - 1].x : 0xFFFFFFFFu;
    if (key >= p.vocab || following != key) return;       // nothing goes on
    if (first == key && earlier == key) return;           // the chain started earlier
    const uint32_t third = p.pairs[min(piece + 2, p.pieces - 1) * p.piece].x;
    const bool longer = piece + 2 < p.pieces && third == key;
    const int group = threadIdx.x / groupThreads, groups = 256 / groupThreads;
    const int64_t pack = static_cast<int64_t>(blockIdx.y) * groupThreads + threadIdx.x % groupThreads;
    const bool live = pack * kN < p.dim;
    using Part = Pack<float, kN>;
    auto partAt = [&](int64_t row) { return reinterpret_cast<const Part*>(p.ends + row * p.dim)[live ? pack : 0]; };
    float sum[kN] = {};
    if (group == 0) {
        const Part a = partAt(piece * 2 + 1), b = partAt((piece + 1) * 2);
#pragma unroll
        for (int j = 0; j < kN; ++j) sum[j] = a.v[j] + b.v[j];
    }
    if (longer) {
        // batches of parts with the keys that tell how far the chain goes, all loads first; behind the last piece they read
        // that one again
        constexpr int kAhead = 8;
        for (int64_t q = piece + 2 + group * kAhead;; q += groups * kAhead) {
            Part part[kAhead];
            uint32_t keys[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int64_t at = min(q + u, p.pieces - 1);
                keys[u] = p.pairs[at * p.piece].x;
                part[u] = partAt(at * 2);
            }
            // what does not belong is masked out bit by bit: a select would let the loads wait for the comparisons
            uint32_t mask = 0xFFFFFFFFu;
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                mask &= q + u < p.pieces && keys[u] == key ? 0xFFFFFFFFu : 0u;
#pragma unroll
                for (int j = 0; j < kN; ++j) sum[j] += __uint_as_float(__float_as_uint(part[u].v[j]) & mask);
            }
            if (mask == 0) break;
        }
        if (groups > 1) {
#pragma unroll
            for (int j = 0; j < kN; ++j) joined[threadIdx.x * kN + j] = sum[j];
            __syncthreads();
            for (int g = 1; g < groups && group == 0; ++g) {
#pragma unroll
                for (int j = 0; j < kN; ++j) sum[j] += joined[(g * groupThreads + threadIdx.x) * kN + j];
            }
        }
    }
    if (group == 0 && live) storeRow<TOut, kN>(static_cast<TOut*>(p.dtable) + static_cast<int64_t>(key) * p.dim, pack, sum, p.scale, p.accumulate != 0);
}

struct SortPlan {
    int passes, bits, cluster;
};
SortPlan sortPlan(int64_t tokens, int64_t vocab) {
    int width = 1;
    while ((1ll << width) <= vocab) ++width;   // rows 0 .. vocab - 1, and vocab for "none"
    SortPlan s;
    s.passes = (width + kMaxDigitBits - 1) / kMaxDigitBits;
    s.bits = (width + s.passes - 1) / s.passes;
    s.cluster = tokens <= 8192 ? 1 : kSortCluster;   // a block alone needs no cluster barriers and no fences beyond its SM
    return s;
}

struct EmbedWorkspace {
    size_t list, ends, map, total;
    int piece;
    int64_t pieces;
};
// Entries per piece: as many as leave eight blocks for each of 148 SMs (the ends of a piece cost two rows of fp32, so long
// pieces move less), between 8 and 128.
EmbedWorkspace embedWorkspace(int64_t tokens, int64_t vocab, int64_t dim) {
    EmbedWorkspace w;
    const int64_t share = tokens * ((dim + 1023) / 1024) / (148 * 8);
    w.piece = 8;
    while (w.piece * 2 <= std::min<int64_t>(share, kMaxPiece)) w.piece *= 2;
    w.pieces = (tokens + w.piece - 1) / w.piece;
    w.list = static_cast<size_t>(roundUp(std::max<int64_t>(tokens, 1) * 4, 256));
    w.ends = static_cast<size_t>(roundUp(w.pieces * 2 * dim * 4, 256));
    w.map = static_cast<size_t>(roundUp((vocab + 31) / 32 * 4, 256));
    w.total = 4 * w.list + w.ends + w.map;
    return w;
}

template <typename TIn, typename TOut, int kN>
void launchReduce(ReduceParams p, cudaStream_t stream) {
    p.columnBlocks = (p.dim / kN + kReduceThreads - 1) / kReduceThreads;
    const int64_t zeroBlocks = p.accumulate ? 0 : (p.vocab + kZeroRows - 1) / kZeroRows;
    const int64_t blocks = p.pieces * p.columnBlocks + zeroBlocks;
    if (blocks > 0) {
        launchDependent(embedReduceKernel<TIn, TOut, kN>, dim3(static_cast<unsigned>(blocks)), dim3(kReduceThreads), 0, stream, p);
        BFB_LAUNCH_CHECK();
        noteLaunch();
    }
    if (p.pieces > 1) {
        constexpr int kJoin = kN == 1 ? 1 : 4;
        const int64_t packs = (p.dim + kJoin - 1) / kJoin;
        int groupThreads = 32;
        // Four columns a thread in four groups or more, or one in as few blocks as hold the row. Measured (2B-class / 10007 x 1001
        // bf16 case): 64 threads a group 19 / 24 us, 256 36 / 15 us.
        const int widest = kJoin == 4 ? 64 : 256;
        while (groupThreads < widest && groupThreads < packs) groupThreads *= 2;
        const dim3 grid(static_cast<unsigned>(p.pieces - 1), static_cast<unsigned>((packs + groupThreads - 1) / groupThreads));
        launchDependent(embedJoinKernel<TOut, kJoin>, grid, dim3(256), 0, stream, p, groupThreads);
        BFB_LAUNCH_CHECK();
        noteLaunch();
    }
}

template <typename TIn, typename TOut>
void reduceAnyPack(const ReduceParams& p, cudaStream_t stream) {
    constexpr int kWide = 16 / static_cast<int>(sizeof(TIn));
    const bool wide = p.dim % kWide == 0 && p.ldDout % kWide == 0 && aligned16(p.dout) && aligned16(p.dtable) && p.dim * sizeof(TOut) % 16 == 0;
    if (wide) launchReduce<TIn, TOut, kWide>(p, stream);
    else launchReduce<TIn, TOut, 1>(p, stream);
}

template <typename TIn, typename TOut>
void launchLookup(const float* ids, const void* table, void* out, int64_t ldOut, int64_t tokens, int64_t vocab, int64_t dim, float scale,
                  int* oobCount, cudaStream_t stream) {
    constexpr int kWide = sizeof(TIn) == 2 && sizeof(TOut) == 2 ? 8 : 4;
    const bool wide = dim % kWide == 0 && ldOut % kWide == 0 && aligned16(table) && aligned16(out);
    const int64_t packs = wide ? dim / kWide : dim;
    const int across = static_cast<int>(std::min<int64_t>(256, roundUp(packs, 32)));
    const dim3 block(across, 256 / across);
    const int64_t blocks = (tokens + static_cast<int64_t>(block.y) * kTokens - 1) / (static_cast<int64_t>(block.y) * kTokens);
    const int grid = static_cast<int>(std::min<int64_t>(blocks, static_cast<int64_t>(smCount()) * 32));
    const auto* t = static_cast<const TIn*>(table);
    auto* o = static_cast<TOut*>(out);
    if (wide) embedScaledKernel<TIn, TOut, kWide><<<grid, block, 0, stream>>>(ids, t, o, ldOut, tokens, vocab, dim, scale, oobCount);
    else embedScaledKernel<TIn, TOut, 1><<<grid, block, 0, stream>>>(ids, t, o, ldOut, tokens, vocab, dim, scale, oobCount);
    BFB_LAUNCH_CHECK();
    noteLaunch();
}

void checkSizes(int64_t tokens, int64_t vocab, int64_t dim) {
    require(tokens >= 0 && vocab > 0 && dim > 0, "embed_scaled: sizes must be positive");
    require(tokens < (1ll << 31) && vocab <= (1ll << 24) && dim <= (1ll << 20), "embed_scaled: sizes beyond the limits (2^31 tokens, 2^24 rows, 2^20 columns)");
}

}  // namespace

void embedScaled(const float* ids, const void* table, int tableDtype, void* out, int outDtype, int64_t ldOut, int64_t tokens, int64_t vocab,
                 int64_t dim, float scale, int* oobCount, cudaStream_t stream) {
    checkSizes(tokens, vocab, dim);
    require(tableDtype == BFB_F32 || tableDtype == BFB_BF16, "embed_scaled: the table must be f32 or bf16");
    require(outDtype == BFB_F32 || outDtype == BFB_BF16, "embed_scaled: the output must be f32 or bf16");
    require(ldOut >= dim, "embed_scaled: row pitch smaller than dim");
    if (tokens == 0) return;
    require(ids != nullptr && table != nullptr && out != nullptr, "embed_scaled: null pointer");
    using bf = __nv_bfloat16;
    if (tableDtype == BFB_F32) {
        if (outDtype == BFB_F32) launchLookup<float, float>(ids, table, out, ldOut, tokens, vocab, dim, scale, oobCount, stream);
        else launchLookup<float, bf>(ids, table, out, ldOut, tokens, vocab, dim, scale, oobCount, stream);
    } else {
        if (outDtype == BFB_F32) launchLookup<bf, float>(ids, table, out, ldOut, tokens, vocab, dim, scale, oobCount, stream);
        else launchLookup<bf, bf>(ids, table, out, ldOut, tokens, vocab, dim, scale, oobCount, stream);
    }
}

size_t embedScaledBackwardWorkspaceBytes(int64_t tokens, int64_t vocab, int64_t dim) {
    checkSizes(tokens, vocab, dim);
    return embedWorkspace(tokens, vocab, dim).total;
}

void embedScaledBackward(const float* ids, const void* dout, int doutDtype, int64_t ldDout, void* dtable, int dtableDtype, int64_t tokens,
                         int64_t vocab, int64_t dim, float scale, bool accumulate, void* workspace, size_t workspaceBytes,
                         cudaStream_t stream) {
    checkSizes(tokens, vocab, dim);
    require(doutDtype == BFB_F32 || doutDtype == BFB_BF16, "embed_scaled_bwd: the gradient must be f32 or bf16");
    require(dtableDtype == BFB_F32 || dtableDtype == BFB_BF16, "embed_scaled_bwd: the table's gradient must be f32 or bf16");
    require(ldDout >= dim, "embed_scaled_bwd: row pitch smaller than dim");
    require(dtable != nullptr, "embed_scaled_bwd: null pointer");
    if (tokens > 0) require(ids != nullptr && dout != nullptr, "embed_scaled_bwd: null pointer");
    const EmbedWorkspace need = embedWorkspace(tokens, vocab, dim);
    require(tokens == 0 || (workspace != nullptr && workspaceBytes >= need.total && reinterpret_cast<uintptr_t>(workspace) % 256 == 0),
            "embed_scaled_bwd: the workspace is missing, too small (bfb_embed_scaled_bwd_workspace) or not 256-byte aligned");
    ReduceParams p{};
    p.count = tokens;
    p.vocab = vocab;
    p.dim = dim;
    p.dout = dout;
    p.ldDout = ldDout;
    p.dtable = dtable;
    p.scale = scale;
    p.accumulate = accumulate ? 1 : 0;
    p.piece = need.piece;
    p.pieces = need.pieces;
    if (tokens > 0) {
        auto* base = static_cast<uint8_t*>(workspace);
        SortBuffers buf;
        for (int i = 0; i < 2; ++i) buf.pairs[i] = reinterpret_cast<uint2*>(base + 2 * i * need.list);
        p.ends = reinterpret_cast<float*>(base + 4 * need.list);
        auto* occurs = reinterpret_cast<uint32_t*>(base + 4 * need.list + need.ends);
        p.occurs = occurs;
        const SortPlan s = sortPlan(tokens, vocab);
        p.pairs = buf.pairs[(s.passes - 1) & 1];
        const size_t smem = static_cast<size_t>(kSortWarps + 2) * (1u << s.bits) * 4;
        BFB_CUDA(cudaFuncSetAttribute(sortTokensKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(static_cast<unsigned>(s.cluster));
        cfg.blockDim = dim3(kSortThreads);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = stream;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = static_cast<unsigned>(s.cluster);
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        BFB_CUDA(cudaLaunchKernelEx(&cfg, sortTokensKernel, ids, buf, occurs, tokens, vocab, s.passes, s.bits, s.cluster));
        noteLaunch();
    }
    using bf = __nv_bfloat16;
    if (doutDtype == BFB_F32) {
        if (dtableDtype == BFB_F32) reduceAnyPack<float, float>(p, stream);
        else reduceAnyPack<float, bf>(p, stream);
    } else {
        if (dtableDtype == BFB_F32) reduceAnyPack<bf, float>(p, stream);
        else reduceAnyPack<bf, bf>(p, stream);
    }
}

}  // namespace bfb
