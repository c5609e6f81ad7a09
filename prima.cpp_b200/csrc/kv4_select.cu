// prima.cpp_b200/csrc/kv4_select.cu — which cells of a sequence stay: the first few, the last few, and of those between the ones with the largest sums of weights.
//
// Mathematics.  A sum becomes a key whose order as a whole number is that of the sums; the need-th largest key is found digit by digit (11, 11, 10 bits): a histogram of the keys that agree with
// the digits so far, and from its top the digit at which the count passes what is needed.  Larger keys stay, of equal ones the lowest cells.  A running count gives each its place.
// A cluster has a sequence, a CTA of it a contiguous part, whose keys stay in shared memory: sums are read once.  Histograms are added up over the cluster through shared memory.
#include <cuda_runtime.h>

#include <atomic>
#include <climits>

#include "../../include/prima_b200.h"
#include "cluster.cuh"
#include "launch.h"

extern std::atomic<uint64_t> g_launches;

namespace pb {
namespace {

constexpr int KS_THREADS = 512, KS_BINS = 2048, KS_TILE = 4 * KS_THREADS;
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
    uint32_t bins[3][KS_BINS];
    int warp[KS_THREADS / 32];
    int counts[2];             // what the other CTAs read: cells that stay for sure, and those at the border
    int digit, above;
};

// keys in the order of the sums; a sum that is no number counts as -inf, -0 as 0
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x == x ? x + 0.f : -INFINITY);
    return u >> 31 ? ~u : u | 0x80000000u;
}
// sum over the threads in front of this one; all: over all of them
__device__ __forceinline__ int in_front(int x, int * warps, int & all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int upto = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
    }
    __syncthreads();
    if (lane == 31) warps[warp] = upto;
    __syncthreads();
    int before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < KS_THREADS / 32; w++) {
        const int k = warps[w];
        if (w < warp) before += k;
        all += k;
    }
    return before + upto - x;
}

template <bool HELD>
__global__ void __launch_bounds__(KS_THREADS) k_kv4_select(const __grid_constant__ Kv4Select A) {
    extern __shared__ __align__(16) uint32_t held[];
    __shared__ __align__(16) KsSmem S;
    const uint32_t rank = cluster_rank(), ctas = cluster_size();
    const int s = blockIdx.x / ctas, tid = threadIdx.x;
    const int len = (int) max((int64_t) 0, min((int64_t) min(A.kv_len[s], A.max_len), A.ld_sums));
    const int count = (int) max((int64_t) 0, min((int64_t) min(A.budget[s], len), A.ld_index));
    const int last = min(A.keep_last, count), first = min(A.keep_first, count - last), end = len - last;      // [first, end): those between
    const int lo = (int) ((int64_t) len * rank / ctas), n = (int) ((int64_t) len * (rank + 1) / ctas) - lo;
    const float * const src = A.sums + s * A.ld_sums + lo;
    int need = count - first - last;
    const bool choose = need > 0 && need < end - first;
    for (int i = tid; i < 3 * KS_BINS; i += KS_THREADS) (&S.bins[0][0])[i] = 0;
    __syncthreads();
    auto key = [&](int i) { return HELD ? held[i] : key_of(src[i]); };
    auto between = [&](int i) { return lo + i >= first && lo + i < end; };
    // all: every key is larger than 0; none: no key is larger than the largest
    uint32_t border = need > 0 ? 0u : 0xffffffffu;
    int of_border = need > 0 ? INT_MAX : 0;          // cells with that key that stay
    if (HELD || choose)
        for (int i = tid; i < n; i += KS_THREADS) {
            const uint32_t k = key_of(src[i]);
            if (HELD) held[i] = k;
            if (choose && between(i)) atomicAdd(&S.bins[0][k >> 21], 1u);
        }
    if (choose) {
        border = 0;
#pragma unroll 1
        for (int pass = 0; pass < 3; pass++) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
            const uint32_t mask = pass == 2 ? 1023u : 2047u;
            if (pass > 0)
                for (int i = tid; i < n; i += KS_THREADS) {
                    const uint32_t k = key(i);
                    if (between(i) && k >> (pass == 1 ? 21 : 10) == border >> (pass == 1 ? 21 : 10)) atomicAdd(&S.bins[pass][k >> shift & mask], 1u);
                }
            cluster_sync();
            // this thread's four bins, from the top
            uint4 c = make_uint4(0u, 0u, 0u, 0u);
            const int b0 = KS_BINS - 4 - 4 * tid;
            for (uint32_t r = 0; r < ctas; r++) {
                const uint4 o = remote(reinterpret_cast<const uint4 *>(&S.bins[pass][b0]), r);
                c.x += o.x; c.y += o.y; c.z += o.z; c.w += o.w;
            }
            const int bin[4] = {(int) c.w, (int) c.z, (int) c.y, (int) c.x};
            int all, above = in_front(bin[0] + bin[1] + bin[2] + bin[3], S.warp, all);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (above < need && need <= above + bin[e]) {
                    S.digit = b0 + 3 - e;
                    S.above = above;
                }
                above += bin[e];
            }
            __syncthreads();
            border |= (uint32_t) S.digit << shift;
            need -= S.above;
        }
        of_border = need;
    } else __syncthreads();
    // 2: stays, 1: at the border
    auto kind = [&](int i) { return !between(i) ? 2 : key(i) > border ? 2 : key(i) == border ? 1 : 0; };
    int mine = 0, at_border = 0;
    for (int i = tid; i < n; i += KS_THREADS) {
        const int k = kind(i);
        mine += k == 2;
        at_border += k == 1;
    }
    int all2, all1;
    in_front(mine, S.warp, all2);
    in_front(at_border, S.warp, all1);
    if (tid == 0) { S.counts[0] = all2; S.counts[1] = all1; }
    cluster_sync();
    int before2 = 0, before1 = 0;
    for (uint32_t r = 0; r < rank; r++) { before2 += remote(&S.counts[0], r); before1 += remote(&S.counts[1], r); }
    if (rank == 0 && tid == 0) A.count[s] = count;
    for (int i0 = 0; i0 < n; i0 += KS_TILE) {
        int k[4], two = 0, one = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int i = i0 + 4 * tid + e;
            k[e] = i < n ? kind(i) : 0;
            two += k[e] == 2;
            one += k[e] == 1;
        }
        int all;
        const int f = in_front(two | one << 16, S.warp, all);
        int at2 = before2 + (f & 0xffff), at1 = before1 + (f >> 16);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int i = i0 + 4 * tid + e, to = at2 + min(at1, of_border);
            if (k[e] == 2 || (k[e] == 1 && at1 < of_border)) {
                A.index[s * A.ld_index + to] = lo + i;
                if (A.kept) A.kept[s * A.ld_kept + to] = src[i];
            }
            at2 += k[e] == 2;
            at1 += k[e] == 1;
        }
        before2 += all & 0xffff;
        before1 += all >> 16;
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
    if (n_seq > INT32_MAX / 8) return PB200_ENOTSUP;
    if (n_seq == 0) return 0;
    if (kept) {   // places are written while others are read
        const float * a = sums + (n_seq - 1) * ld_sums + (ld_sums < max_len ? ld_sums : max_len), * b = kept + (n_seq - 1) * ld_kept + (ld_index < max_len ? ld_index : max_len);
        if ((uintptr_t) kept < (uintptr_t) a && (uintptr_t) sums < (uintptr_t) b) return PB200_EINVAL;
    }
    const Kv4Select a{sums, ld_sums, kv_len, budget, max_len, keep_first, keep_last, index, ld_index, count, kept, ld_kept};
    const int64_t most = ld_sums < max_len ? ld_sums : max_len;
    const int ctas = most > 8192 ? 8 : most > 4096 ? 4 : most > 2048 ? 2 : 1;
    const size_t smem = (size_t) (most / ctas + 1) * sizeof(uint32_t);
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
