// prima.cpp_b200/csrc/kv4_select.cu — which cells of a sequence stay: the first few, the last few, and of those between the ones with the largest sums of weights.
//
// Mathematics.  A sum becomes a key whose order as a whole number is that of the sums; the need-th largest key is found digit by digit (8 bits): a histogram of the keys that agree with
// the digits so far, and from its top the digit at which the count passes what is needed.  Larger keys stay, of equal ones the lowest cells.  A running count gives each its place.
// A cluster has a sequence, a CTA of it a contiguous part, whose keys stay in shared memory: sums are read once.  Histograms are added up over the cluster through shared memory.  Cells that no
// query sees have a sum of 0, as often as not most of them: these are counted apart, and added to their bin once a warp.
//
// Bound: the eight CTAs of the longest sequence (a lane has four keys at a time; of the whole GPU issue slots 27 %, DRAM 3 %), the chain of passes, each some 1.3 us for barrier, bins and counts, where it is short.  us, 24 sequences of up to
// 131 072 cells: one key at a time 46 to 49, whether digits have 8 or 11 bits; four at a time 31; kept sums from their keys, not from memory again, 27; clusters of 16 CTAs 42.  1000 cells: 10.
#include <cuda_runtime.h>

#include <atomic>
#include <climits>

#include "../../include/prima_b200.h"
#include "cluster.cuh"
#include "launch.h"

extern std::atomic<uint64_t> g_launches;

namespace pb {
namespace {

constexpr int KS_WARPS = 16, KS_THREADS = 32 * KS_WARPS, KS_BINS = 256, KS_PASSES = 4, KS_CTAS = 8;
constexpr int KS_STEP = 128;                // keys of a warp at a time: four to a lane
constexpr size_t KS_HELD = 192 * 1024;

struct Kv4Select {
    const float * sums;
    int64_t ld_sums;
    const int32_t * kv_len, * budget;
    int max_len, keep_first, keep_last;
    int32_t * index;
    int64_t ld_index;
    int32_t * count;
    float * kept;
    int64_t ld_kept;
};

struct KsSmem {
    uint32_t bins[KS_PASSES][KS_BINS];
    int warp[KS_WARPS], stay[KS_WARPS][2];
    int counts[2];             // what the other CTAs read: cells that stay for sure, and those at the border
    int digit, above;
};

// keys in the order of the sums; a sum that is no number counts as -inf, -0 as 0.  All are larger than 0, which stands for no cell
constexpr uint32_t ZERO_KEY = 0x80000000u, LEAST_KEY = 0x007fffffu, ALWAYS = 0xffffffffu;      // of a sum of 0, of -inf, of the cells that stay whatever their sums
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x == x ? x + 0.f : -INFINITY);
    return u ^ ((uint32_t) ((int32_t) u >> 31) | 0x80000000u);
}
__device__ __forceinline__ int upto(int x) {              // sum over the lanes up to this one
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    return x;
}
// sum over the threads in front of this one; all: over all of them
__device__ __forceinline__ int in_front(int x, int * warps, int & all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, mine = upto(x);
    __syncthreads();
    if (lane == 31) warps[warp] = mine;
    __syncthreads();
    const int ends = upto(lane < KS_WARPS ? warps[lane % KS_WARPS] : 0), before = __shfl_sync(0xffffffffu, ends, (warp + 31) % 32);
    all = __shfl_sync(0xffffffffu, ends, 31);
    return (warp > 0 ? before : 0) + mine - x;
}
template <bool HELD>
__global__ void __launch_bounds__(KS_THREADS) k_kv4_select(const __grid_constant__ Kv4Select A) {
    extern __shared__ __align__(16) uint32_t held[];
    __shared__ __align__(16) KsSmem S;
    const uint32_t rank = cluster_rank(), ctas = cluster_size();
    const int s = blockIdx.x / ctas, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int len = (int) max((int64_t) 0, min((int64_t) min(A.kv_len[s], A.max_len), A.ld_sums));
    const int count = (int) max((int64_t) 0, min((int64_t) min(A.budget[s], len), A.ld_index));
    const int last = min(A.keep_last, count), first = min(A.keep_first, count - last), end = len - last;      // [first, end): those between
    const int lo = (int) ((int64_t) len * rank / ctas), n = (int) ((int64_t) len * (rank + 1) / ctas) - lo;
    const float * const src = A.sums + s * A.ld_sums + lo;
    if (tid < KS_BINS)
#pragma unroll
        for (int p = 0; p < KS_PASSES; p++) S.bins[p][tid] = 0;
    // a warp has a contiguous part of the CTA's, whole steps, and shared memory for them
    const int per = (n + KS_WARPS * KS_STEP - 1) / (KS_WARPS * KS_STEP) * KS_STEP, s0 = min(n, warp * per), s1 = min(n, s0 + per);
    auto key_at = [&](int i, float x) { return i >= n ? 0u : lo + i < first || lo + i >= end ? ALWAYS : key_of(x); };
    auto four = [&](int i) {                         // keys of the cells i .. i + 3
        if (HELD) return *reinterpret_cast<const uint4 *>(held + i);
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = i + e < n ? src[i + e] : 0.f;
        return make_uint4(key_at(i, x[0]), key_at(i + 1, x[1]), key_at(i + 2, x[2]), key_at(i + 3, x[3]));
    };
    if (HELD) {   // all of the sums on their way at once
        for (int i = s0 + lane; i < s1; i += 32) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(&held[i])), "l"(src + i) : "memory");
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();                                // (a warp reads its own)
    }
    __syncthreads();
    // all stay: every key is larger than 0; only those that stay anyway are larger than the last but one; otherwise the border is looked for
    const bool choose = count - first - last > 0 && count < len;
    uint32_t border = count == len ? 0u : ALWAYS - 1;
    int of_border = 0, need = count;                 // cells with that key that stay; how many are to be found
    if (HELD || choose) {
        int zeros = 0;
        for (int i = s0 + 4 * lane; i - 4 * lane < s1; i += KS_STEP) {
            uint4 v = HELD ? *reinterpret_cast<const uint4 *>(held + i) : four(i);
            uint32_t k[4] = {v.x, v.y, v.z, v.w};
            if (HELD) {
                const int at = lo + i - 4 * lane;    // the step's first cell
                if (at >= first && at + KS_STEP <= end && i - 4 * lane + KS_STEP <= n)
#pragma unroll
                    for (int e = 0; e < 4; e++) k[e] = key_of(__uint_as_float(k[e]));
                else
#pragma unroll
                    for (int e = 0; e < 4; e++) k[e] = key_at(i + e, __uint_as_float(k[e]));
                *reinterpret_cast<uint4 *>(held + i) = make_uint4(k[0], k[1], k[2], k[3]);
            }
            if (choose)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if (k[e] == ZERO_KEY) zeros++;
                    else atomicAdd(&S.bins[0][k[e] >> 24], 1u);
                }
        }
        if (choose) {
            zeros = __reduce_add_sync(0xffffffffu, zeros);
            if (lane == 0 && zeros) atomicAdd(&S.bins[0][ZERO_KEY >> 24], (uint32_t) zeros);
        }
    }
    if (choose) {
        border = 0;
#pragma unroll 1
        for (int pass = 0; pass < KS_PASSES; pass++) {
            const int shift = 24 - 8 * pass;
            if (pass > 0) {
                int zeros = 0;
                const uint32_t width = 1u << (shift + 8);                 // keys that agree so far: border .. border + width - 1
                for (int i = s0 + 4 * lane; i - 4 * lane < s1; i += KS_STEP) {
                    const uint4 v = four(i);
                    const uint32_t k[4] = {v.x - border, v.y - border, v.z - border, v.w - border};
                    if (k[0] < width || k[1] < width || k[2] < width || k[3] < width)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (k[e] < width) {
                                if (k[e] + border == ZERO_KEY) zeros++;
                                else atomicAdd(&S.bins[pass][k[e] >> shift], 1u);
                            }
                }
                zeros = __reduce_add_sync(0xffffffffu, zeros);
                if (lane == 0 && zeros) atomicAdd(&S.bins[pass][ZERO_KEY - border >> shift], (uint32_t) zeros);
            }
            cluster_sync();
            // a thread has a bin of all CTAs, from the top
            int of[KS_CTAS], bin = 0;
            const int b = KS_BINS - 1 - tid;
#pragma unroll
            for (int r = 0; r < KS_CTAS; r++) of[r] = b >= 0 && r < (int) ctas ? remote(reinterpret_cast<const int *>(&S.bins[pass][b]), r) : 0;
#pragma unroll
            for (int r = 0; r < KS_CTAS; r++) bin += of[r];
            int all;
            const int above = in_front(bin, S.warp, all);
            if (above < need && need <= above + bin) {
                S.digit = b;
                S.above = above;
            }
            __syncthreads();
            border |= (uint32_t) S.digit << shift;
            need -= S.above;
        }
        of_border = need;
    }
    // those that stay, and those at the border
    int stay[2] = {0, 0};
    for (int i = s0 + 4 * lane; i - 4 * lane < s1; i += KS_STEP) {
        const uint4 v = four(i);
        stay[0] += (v.x > border) + (v.y > border) + (v.z > border) + (v.w > border);
        stay[1] += (v.x == border) + (v.y == border) + (v.z == border) + (v.w == border);
    }
    stay[0] = __reduce_add_sync(0xffffffffu, stay[0]);
    stay[1] = __reduce_add_sync(0xffffffffu, stay[1]);
    if (lane < 2) S.stay[warp][lane] = stay[lane & 1];
    __syncthreads();
    int before[2], all[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
        const int ends = upto(lane < KS_WARPS ? S.stay[lane % KS_WARPS][e] : 0), front = __shfl_sync(0xffffffffu, ends, (warp + 31) % 32);
        before[e] = warp > 0 ? front : 0;
        all[e] = __shfl_sync(0xffffffffu, ends, 31);
    }
    if (tid < 2) S.counts[tid] = all[tid & 1];
    cluster_sync();
    {
        int of[KS_CTAS][2];
#pragma unroll
        for (int r = 0; r < KS_CTAS; r++)
#pragma unroll
            for (int e = 0; e < 2; e++) of[r][e] = r < (int) rank ? remote(&S.counts[e], r) : 0;
#pragma unroll
        for (int r = 0; r < KS_CTAS; r++) { before[0] += of[r][0]; before[1] += of[r][1]; }
    }
    if (rank == 0 && tid == 0) A.count[s] = count;
    int32_t * const index = A.index + s * A.ld_index;
    float * const kept = A.kept ? A.kept + s * A.ld_kept : nullptr;
    const uint32_t lower = (1u << lane) - 1;
    for (int i = s0 + 4 * lane; i - 4 * lane < s1; i += KS_STEP) {
        const uint4 v = four(i);
        const uint32_t k[4] = {v.x, v.y, v.z, v.w};
        uint32_t over[4], at[4];
        int to = before[0], ties = before[1];        // in front of this lane's
#pragma unroll
        for (int e = 0; e < 4; e++) {
            over[e] = __ballot_sync(0xffffffffu, k[e] > border);
            to += __popc(over[e] & lower);
            before[0] += __popc(over[e]);
        }
        if (__any_sync(0xffffffffu, k[0] == border || k[1] == border || k[2] == border || k[3] == border))
#pragma unroll
            for (int e = 0; e < 4; e++) {
                at[e] = __ballot_sync(0xffffffffu, k[e] == border);
                ties += __popc(at[e] & lower);
                before[1] += __popc(at[e]);
            }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const bool tie = k[e] == border;
            if (k[e] > border || (tie && ties < of_border)) {
                const int place = to + min(ties, of_border);
                index[place] = lo + i + e;
                // a key gives its sum back, but for those that may come from several
                if (kept) kept[place] = k[e] == ALWAYS || k[e] == ZERO_KEY || k[e] == LEAST_KEY ? src[i + e] : __uint_as_float(k[e] ^ (k[e] >> 31 ? 0x80000000u : 0xffffffffu));
            }
            to += k[e] > border;
            ties += tie;
        }
    }
    cluster_sync();                                  // nobody reads a CTA's numbers that has ended
}

}  // namespace
}  // namespace pb

using namespace pb;

extern "C" int pb200_kv4_select(int n_seq, const float * sums, int64_t ld_sums, const int32_t * kv_len, int max_len, const int32_t * budget, int keep_first, int keep_last, int32_t * index,
                                int64_t ld_index, int32_t * count, float * kept, int64_t ld_kept, void * stream) {
    if (n_seq < 0 || max_len < 0 || keep_first < 0 || keep_last < 0 || !sums || ld_sums <= 0 || !kv_len || !budget || !index || ld_index <= 0 || !count) return PB200_EINVAL;
    if (((uintptr_t) sums & 3) || (kept && (((uintptr_t) kept & 3) || ld_kept < (ld_index < max_len ? ld_index : max_len)))) return PB200_EINVAL;
    if (n_seq > INT32_MAX / KS_CTAS) return PB200_ENOTSUP;
    if (n_seq == 0) return 0;
    if (kept) {   // places are written while others are read
        const float * a = sums + (n_seq - 1) * ld_sums + (ld_sums < max_len ? ld_sums : max_len), * b = kept + (n_seq - 1) * ld_kept + (ld_index < max_len ? ld_index : max_len);
        if ((uintptr_t) kept < (uintptr_t) a && (uintptr_t) sums < (uintptr_t) b) return PB200_EINVAL;
    }
    const Kv4Select a{sums, ld_sums, kv_len, budget, max_len, keep_first, keep_last, index, ld_index, count, kept, ld_kept};
    const int64_t most = ld_sums < max_len ? ld_sums : max_len;
    const int ctas = most > 8192 ? KS_CTAS : most > 4096 ? 4 : most > 2048 ? 2 : 1;
    const size_t smem = (size_t) (most / ctas + 1 + KS_WARPS * KS_STEP - 1) / (KS_WARPS * KS_STEP) * (KS_WARPS * KS_STEP) * sizeof(uint32_t);
    const bool hold = smem <= KS_HELD;
    if (hold) {
        static FuncAttrCache cache;
        const cudaError_t e = ensure_dyn_smem(cache, (const void *) k_kv4_select<true>, KS_HELD, false);
        if (e != cudaSuccess) return (int) e;
    }
    const cudaStream_t st = (cudaStream_t) stream;
    const cudaError_t e = hold ? launch_clusters(k_kv4_select<true>, n_seq, ctas, KS_THREADS, smem, false, st, a) : launch_clusters(k_kv4_select<false>, n_seq, ctas, KS_THREADS, 0, false, st, a);
    if (e == cudaSuccess) g_launches++;
    return (int) e;
}
