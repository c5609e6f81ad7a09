// prima.cpp_b200/csrc/verify.cu — verification of drafted tokens: how many of a sequence's drafts the target accepts, and the token that follows them.
//
// Mathematics.  With p and q the softmax of the target's and the draft's logits times t = 1 / temperature, drafted token x is accepted where u q(x) < p(x).  Behind the accepted ones comes a
// token from max(p - q, 0) at the place of the rejection, from p behind the last draft: by the inverse of the cumulative sum at v times the whole.  What is emitted then has the target's
// distribution, whatever the draft's.
//   rows    a CTA has a chunk of a row: its largest logit m and the sum of 2^((l - m) t log2 e), in 32 bits: a decision u q < p changes where they are within 1e-7 of each other
//   draw    a cluster has a sequence.  It joins its rows' chunks, decides, and takes the one row (two, with draft logits) that the token is drawn from into shared memory.  Weights and sums are in
//           64 bits: a cumulative sum of 100 000 weights with errors of 1e-8 each would give another token once in a thousand draws.  A row's sum is that of its tiles, of which one is scanned.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cfloat>
#include <climits>

#include "../../include/prima_b200.h"
#include "cluster.cuh"
#include "launch.h"

extern std::atomic<uint64_t> g_launches;

namespace pb {
namespace {

constexpr int VR_THREADS = 256, VR_ONCE = 4;           // rows: vectors of 16 bytes to a thread on their way
constexpr int VD_THREADS = 512, VD_EACH = 4, VD_TILE = VD_THREADS * VD_EACH, VD_TILES = 64;
constexpr size_t VD_SMEM = 220 * 1024;

struct Verify {
    const void * target, * draft;
    int64_t ld_target, ld_draft;
    int vocab, n_seq;
    const int32_t * start;
    int64_t n_drafts;
    const int32_t * tokens;
    const float * inv_temp, * u, * v;
    int32_t * accepted, * out;
    int64_t ld_out;
    const int32_t * kv_len;
    int32_t * kv_len_out;
    float4 * parts;            // [2][n_drafts][chunks]: largest logit, sum of weights, index of the largest (bits)
    int chunks;
};

__device__ __forceinline__ float number(float x) { return fmaxf(x, -INFINITY); }      // a logit that is none counts as -inf
__device__ __forceinline__ float get(const float * p) { return number(*p); }
__device__ __forceinline__ float get(const __half * p) { return number(__half2float(*p)); }
__device__ __forceinline__ float get(const __nv_bfloat16 * p) { return number(__bfloat162float(*p)); }
template <typename T> constexpr int vec() { return 16 / (int) sizeof(T); }
// vector v of a row of n: entries v * vec - skew and on, those outside -inf.  skew: entries between a 16-byte boundary and the row's first
template <typename T>
__device__ __forceinline__ void get_vec(const T * row, int n, int skew, int v, float (&x)[vec<T>()]) {
    const int at = v * vec<T>() - skew;
    if (at >= 0 && at + vec<T>() <= n) {
        const uint4 w = __ldg(reinterpret_cast<const uint4 *>(row + at));
        const T * e = reinterpret_cast<const T *>(&w);
#pragma unroll
        for (int i = 0; i < vec<T>(); i++) x[i] = get(e + i);
    } else {
#pragma unroll
        for (int i = 0; i < vec<T>(); i++) x[i] = at + i >= 0 && at + i < n ? get(row + at + i) : -INFINITY;
    }
}
template <typename T> __device__ __forceinline__ int skew_of(const T * row) { return (int) (((uintptr_t) row & 15) / sizeof(T)); }

// 1 / temperature of a sequence: of 0 the smallest number, so that times -inf it is no NaN; none where it is below 0 or no number
__device__ __forceinline__ float inv_temp_of(const Verify & A, int s) {
    const float t = A.inv_temp ? A.inv_temp[s] : 1.f;
    return t == 0.f ? 1.4e-45f : t;
}

// which sequence draft i belongs to (-1: none), by all threads of a CTA
template <int THREADS>
__device__ __forceinline__ int sequence_of(const Verify & A, int64_t i) {
    int s = 0;
    for (int at = 0; at < A.n_seq; at += THREADS) {
        const int k = at + (int) threadIdx.x;
        s += __syncthreads_count(k < A.n_seq && A.start[k + 1] <= i);
    }
    return s < A.n_seq && A.start[s] <= i && i < A.start[s + 1] ? s : -1;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// sums of weights relative to the largest logit
struct Sum {
    float m = -INFINITY, l = 0.f;
    __device__ __forceinline__ void add(float m2, float l2, float c) {       // c: of a logit to the power of two
        const float top = fmaxf(m, m2);
        if (top == INFINITY) l = (m == INFINITY ? l : 0.f) + (m2 == INFINITY ? l2 : 0.f);
        else if (top > -INFINITY) l = l * ex2((m - top) * c) + l2 * ex2((m2 - top) * c);
        m = top;
    }
};

template <typename T>
__global__ void __launch_bounds__(VR_THREADS) k_verify_rows(const __grid_constant__ Verify A) {
    constexpr int VEC = vec<T>();
    const int64_t row = blockIdx.x / A.chunks;
    const int chunk = (int) (blockIdx.x - row * A.chunks), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const bool of_draft = row >= A.n_drafts;
    const int64_t i = of_draft ? row - A.n_drafts : row;
    pdl_trigger();
    const int s = sequence_of<VR_THREADS>(A, i);
    if (s < 0) return;
    const T * src = of_draft ? (const T *) A.draft + i * A.ld_draft : (const T *) A.target + (i + s) * A.ld_target;
    const int skew = skew_of(src), vecs = (A.vocab + skew + VEC - 1) / VEC;
    const int from = (int) ((int64_t) vecs * chunk / A.chunks), to = (int) ((int64_t) vecs * (chunk + 1) / A.chunks);
    const float t = inv_temp_of(A, s), c = t * 1.4426950408889634f;
    Sum sum;
    int arg = INT_MAX;
    const bool greedy = t == INFINITY;
    for (int v0 = from + tid; v0 < to; v0 += VR_ONCE * VR_THREADS) {
        float x[VR_ONCE][VEC], top = -INFINITY;
#pragma unroll
        for (int k = 0; k < VR_ONCE; k++) {
            if (v0 + k * VR_THREADS < to) get_vec(src, A.vocab, skew, v0 + k * VR_THREADS, x[k]);
            else
#pragma unroll
                for (int e = 0; e < VEC; e++) x[k][e] = -INFINITY;
        }
#pragma unroll
        for (int k = 0; k < VR_ONCE; k++)
#pragma unroll
            for (int e = 0; e < VEC; e++) top = fmaxf(top, x[k][e]);
        if (greedy) {
            if (top > sum.m) {
                sum.m = top;
#pragma unroll
                for (int k = VR_ONCE - 1; k >= 0; k--)
#pragma unroll
                    for (int e = VEC - 1; e >= 0; e--)
                        if (x[k][e] == top) arg = (v0 + k * VR_THREADS) * VEC - skew + e;
            }
        } else if (top > -INFINITY) {
            float l = 0.f;
#pragma unroll
            for (int k = 0; k < VR_ONCE; k++)
#pragma unroll
                for (int e = 0; e < VEC; e++) l += top == INFINITY ? (x[k][e] == INFINITY ? 1.f : 0.f) : ex2((x[k][e] - top) * c);
            sum.add(top, l, c);
        }
    }
    __shared__ Sum sums[VR_THREADS / 32];
    __shared__ int args[VR_THREADS / 32];
    auto join = [&](float m2, float l2, int arg2) {
        if (greedy) {
            if (m2 > sum.m || (m2 == sum.m && arg2 < arg)) { sum.m = m2; arg = arg2; }
        } else sum.add(m2, l2, c);
    };
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, sum.m, o), l2 = __shfl_xor_sync(0xffffffffu, sum.l, o);
        const int arg2 = __shfl_xor_sync(0xffffffffu, arg, o);
        join(m2, l2, arg2);
    }
    if (lane == 0) { sums[warp] = sum; args[warp] = arg; }
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < VR_THREADS / 32; w++) join(sums[w].m, sums[w].l, args[w]);
        A.parts[row * A.chunks + chunk] = make_float4(sum.m, sum.l, __int_as_float(arg), 0.f);
    }
}

struct VdSmem {
    double warp[VD_THREADS / 32][2];
    double mine[8];            // what the other CTAs read: largest logits, indices, sums
    double tile[2][VD_TILES];
    int first, found;
};

// p(x) of a row from its chunks, by a warp
__device__ __forceinline__ double chance(const float4 * parts, int chunks, int x, float lx, float t) {
    const int lane = threadIdx.x & 31;
    float m = -INFINITY;
    for (int k = lane; k < chunks; k += 32) m = fmaxf(m, __ldcg(&parts[k]).x);
    m = warp_max(m);
    if (m == -INFINITY || !(t >= 0.f)) return 0.0;
    if (t == INFINITY) {
        int arg = INT_MAX;
        for (int k = lane; k < chunks; k += 32) {
            const float4 p = __ldcg(&parts[k]);
            if (p.x == m) arg = min(arg, __float_as_int(p.z));
        }
        return __reduce_min_sync(0xffffffffu, arg) == x ? 1.0 : 0.0;
    }
    double l = 0.0;
    for (int k = lane; k < chunks; k += 32) {
        const float4 p = __ldcg(&parts[k]);
        l += m == INFINITY ? (p.x == INFINITY ? p.y : 0.0) : p.y * exp(((double) p.x - m) * t);
    }
    l = warp_sum_d(l);
    return (m == INFINITY ? (lx == INFINITY ? 1.0 : 0.0) : exp(((double) lx - m) * t)) / l;
}

template <typename T, bool HELD>     // HELD: the rows lie in shared memory
__global__ void __launch_bounds__(VD_THREADS) k_verify_draw(const __grid_constant__ Verify A) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    __shared__ VdSmem S;
    float * const held = reinterpret_cast<float *>(smem_raw);
    const uint32_t rank = cluster_rank(), ctas = cluster_size();
    const int s = blockIdx.x / ctas, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // this CTA's tiles of the vocabulary: as many to each
    const int tiles = (A.vocab + VD_TILE - 1) / VD_TILE, t0 = (int) ((int64_t) tiles * rank / ctas), t1 = (int) ((int64_t) tiles * (rank + 1) / ctas);
    const int base = t0 * VD_TILE, n = max(0, min(A.vocab, t1 * VD_TILE) - base);
    const int64_t a = A.start[s], b = A.start[s + 1];
    const bool good = a >= 0 && b >= a && b <= A.n_drafts;
    const int drafts = good ? (int) (b - a) : 0;
    const float t = inv_temp_of(A, s);
    if (tid == 0) S.first = drafts;
    __syncthreads();
    pdl_wait();                                             // the rows' sums
    if (good)
        for (int i = warp; i < drafts; i += VD_THREADS / 32) {
            const int64_t d = a + i;
            const int x = A.tokens[d];
            bool ok = false;
            if (x >= 0 && x < A.vocab) {
                const double p = chance(A.parts + d * A.chunks, A.chunks, x, get((const T *) A.target + (d + s) * A.ld_target + x), t);
                const double q = A.draft ? chance(A.parts + (A.n_drafts + d) * A.chunks, A.chunks, x, get((const T *) A.draft + d * A.ld_draft + x), t) : 1.0;
                ok = (double) A.u[d] * q < p;
            }
            if (!ok && lane == 0) atomicMin(&S.first, i);
        }
    __syncthreads();
    const int acc = S.first;
    if (!good) return;                                      // (all CTAs of the cluster)
    const bool rejected = acc < drafts, two = rejected && A.draft;
    const int out_of = rejected && !A.draft ? A.tokens[a + acc] : -1;       // a token whose weight is 0
    const T * const row_p = (const T *) A.target + (a + s + acc) * A.ld_target, * const row_q = two ? (const T *) A.draft + (a + acc) * A.ld_draft : nullptr;

    // ---- the rows, and their largest logits ----
    auto block_max = [&](float & x, float & y) {
        x = warp_max(x);
        y = warp_max(y);
        if (lane == 0) { S.warp[warp][0] = x; S.warp[warp][1] = y; }
        __syncthreads();
        for (int w = 0; w < VD_THREADS / 32; w++) { x = fmaxf(x, (float) S.warp[w][0]); y = fmaxf(y, (float) S.warp[w][1]); }
        __syncthreads();
    };
    float m[2] = {-INFINITY, -INFINITY};
    int arg = INT_MAX;
    auto take = [&](const T * row, float * to, float & top) {
        constexpr int VEC = vec<T>();
        const T * src = row + base;
        const int skew = skew_of(src), vecs = n > 0 ? (n + skew + VEC - 1) / VEC : 0;
        for (int v0 = tid; v0 < vecs; v0 += 4 * VD_THREADS) {
            float x[4][VEC];
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (v0 + k * VD_THREADS < vecs) get_vec(src, n, skew, v0 + k * VD_THREADS, x[k]);
                else
#pragma unroll
                    for (int e = 0; e < VEC; e++) x[k][e] = -INFINITY;
#pragma unroll
            for (int k = 0; k < 4; k++)
#pragma unroll
                for (int e = 0; e < VEC; e++) {
                    const int at = (v0 + k * VD_THREADS) * VEC - skew + e;
                    if (at < 0 || at >= n) continue;
                    if (x[k][e] > top) {
                        top = x[k][e];
                        if (row == row_p) arg = base + at;
                    }
                    if (HELD) to[at] = x[k][e];
                }
        }
    };
    const int room = (n + 3) & ~3;
    take(row_p, held, m[0]);
    const float mine = m[0];
    if (two) take(row_q, held + room, m[1]);
    block_max(m[0], m[1]);
    if (t == INFINITY) {       // the first of the largest: (that of a thread is the first of its own)
        int first = mine == m[0] ? arg : INT_MAX;
        first = __reduce_min_sync(0xffffffffu, first);
        if (lane == 0) S.warp[warp][0] = first;
        __syncthreads();
        for (int w = 0; w < VD_THREADS / 32; w++) first = min(first, (int) S.warp[w][0]);
        arg = first;
    }
    if (tid == 0) { S.mine[0] = m[0]; S.mine[1] = m[1]; S.mine[2] = arg; }
    cluster_sync();
    int first = INT_MAX;
    for (uint32_t r = 0; r < ctas; r++) { m[0] = fmaxf(m[0], (float) remote(&S.mine[0], r)); m[1] = fmaxf(m[1], (float) remote(&S.mine[1], r)); }
    for (uint32_t r = 0; r < ctas; r++)
        if ((float) remote(&S.mine[0], r) == m[0]) first = min(first, (int) remote(&S.mine[2], r));
    auto finish = [&](int token) {                          // by one thread of the cluster
        if (acc < A.ld_out) A.out[s * A.ld_out + acc] = token;
    };
    if (rank == 0) {
        for (int64_t i = tid; i < acc && i < A.ld_out; i += VD_THREADS) A.out[s * A.ld_out + i] = A.tokens[a + i];
        if (tid == 0) {
            A.accepted[s] = acc;
            if (A.kv_len) A.kv_len_out[s] = A.kv_len[s] - (drafts - acc);
        }
    }
    if (m[0] == -INFINITY || !(t >= 0.f) || t == INFINITY) {       // no weights; all of it on one
        if (rank == 0 && tid == 0) finish(m[0] == -INFINITY || !(t >= 0.f) ? -1 : first);
        cluster_sync();                                     // (the others read this CTA's numbers)
        return;
    }

    // ---- weights ----
    auto weight = [&](float x, float top) { return top == INFINITY ? (x == INFINITY ? 1.0 : 0.0) : exp(((double) x - top) * t); };
    auto load = [&](int which, int i) {                     // logit i of this CTA's
        if (HELD) return held[which * room + i];
        return get((which ? row_q : row_p) + base + i);
    };
    auto block_sum = [&](double & x, double & y) {
        x = warp_sum_d(x);
        y = warp_sum_d(y);
        __syncthreads();
        if (lane == 0) { S.warp[warp][0] = x; S.warp[warp][1] = y; }
        __syncthreads();
        x = y = 0.0;
        for (int w = 0; w < VD_THREADS / 32; w++) { x += S.warp[w][0]; y += S.warp[w][1]; }
    };
    double z[2] = {0.0, 0.0};
    const bool residual_q = two && m[1] > -INFINITY;        // (a draft row without a number takes nothing away)
    if (residual_q) {
        for (int i = tid; i < n; i += VD_THREADS) {
            z[0] += weight(load(0, i), m[0]);
            z[1] += weight(load(1, i), m[1]);
        }
        block_sum(z[0], z[1]);
        if (tid == 0) { S.mine[3] = z[0]; S.mine[4] = z[1]; }
        cluster_sync();
        z[0] = z[1] = 0.0;
        for (uint32_t r = 0; r < ctas; r++) { z[0] += remote(&S.mine[3], r); z[1] += remote(&S.mine[4], r); }
    }
    // entry i's weight, of the distribution at hand and of p
    auto entry = [&](int i, bool rest) {
        const double e = weight(load(0, i), m[0]);
        if (!rest) return e;
        if (residual_q) return fmax(e * z[1] - weight(load(1, i), m[1]) * z[0], 0.0);
        return base + i == out_of ? 0.0 : e;
    };
    bool rest = residual_q || out_of >= 0;
    for (;;) {
        double all = 0.0;
        for (int k = 0; k < t1 - t0; k++) {                 // (tiles beyond the first VD_TILES are added to the last)
            double x = 0.0, y = 0.0;
            for (int i = k * VD_TILE + tid; i < min(n, (k + 1) * VD_TILE); i += VD_THREADS) x += entry(i, rest);
            block_sum(x, y);
            if (tid == 0) S.tile[0][min(k, VD_TILES - 1)] = k < VD_TILES ? x : S.tile[0][VD_TILES - 1] + x;
            all += x;
        }
        __syncthreads();
        if (tid == 0) S.mine[rest ? 5 : 6] = all;
        cluster_sync();
        double total = 0.0, front = 0.0;
        for (uint32_t r = 0; r < ctas; r++) total += remote(&S.mine[rest ? 5 : 6], r);
        if (rest && !(total > 0.0)) {                        // nothing is left: from p
            rest = false;
            continue;
        }
        const double x = (double) A.v[s] * total;
        int owner = 0;
        double cum = 0.0;
        // the first CTA whose end lies beyond x; where rounding leaves none, the last that has any
        for (uint32_t r = 0; r < ctas; r++) {
            const double w = remote(&S.mine[rest ? 5 : 6], r);
            if (w > 0.0) {
                owner = (int) r;
                front = cum;
                if (cum + w > x) break;
            }
            cum += w;
        }
        cluster_sync();                                     // nobody reads this CTA's numbers from here on
        if (owner != (int) rank) return;
        // the tile, in the same way
        int tile = 0;
        double before = front;
        cum = front;
        for (int k = 0; k < min(t1 - t0, VD_TILES); k++) {
            const double w = S.tile[0][k];
            if (w > 0.0) {
                tile = k;
                before = cum;
                if (cum + w > x) break;
            }
            cum += w;
        }
        // the entry
        if (tid == 0) { S.first = INT_MAX; S.found = 0; }
        for (int k = tile;; k++) {
            double w[VD_EACH], sum = 0.0;
            const int i0 = k * VD_TILE + tid * VD_EACH;
#pragma unroll
            for (int e = 0; e < VD_EACH; e++) {
                w[e] = i0 + e < n ? entry(i0 + e, rest) : 0.0;
                sum += w[e];
            }
            double upto = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double y = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += y;
            }
            __syncthreads();
            if (lane == 31) S.warp[warp][0] = upto;
            __syncthreads();
            double c = before, end = before;
            for (int j = 0; j < VD_THREADS / 32; j++) {
                if (j < warp) c += S.warp[j][0];
                end += S.warp[j][0];
            }
            c += upto - sum;
#pragma unroll
            for (int e = 0; e < VD_EACH; e++) {
                c += w[e];
                if (w[e] > 0.0) {
                    atomicMax(&S.found, i0 + e);
                    if (c > x) atomicMin(&S.first, i0 + e);
                }
            }
            __syncthreads();
            const bool last = tile < VD_TILES - 1 || k == t1 - t0 - 1;
            if (S.first != INT_MAX || last) {
                if (tid == 0) finish(base + (S.first != INT_MAX ? S.first : S.found));
                return;
            }
            before = end;
        }
    }
}

template <typename T>
int verify_launch(const Verify & A, cudaStream_t st) {
    if (A.n_drafts > 0) {
        const int64_t ctas = A.n_drafts * (A.draft ? 2 : 1) * A.chunks;
        k_verify_rows<T><<<(unsigned) ctas, VR_THREADS, 0, st>>>(A);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return (int) e;
        g_launches++;
    }
    const int tiles = (A.vocab + VD_TILE - 1) / VD_TILE, ctas = tiles >= 8 ? 8 : tiles >= 4 ? 4 : tiles >= 2 ? 2 : 1;
    const size_t rows = (size_t) ((tiles + ctas - 1) / ctas) * VD_TILE * sizeof(float), smem = rows * (A.draft ? 2 : 1);
    const bool held = smem <= VD_SMEM;
    static FuncAttrCache cache[2];
    const void * fn = held ? (const void *) k_verify_draw<T, true> : (const void *) k_verify_draw<T, false>;
    cudaError_t e = ensure_dyn_smem(cache[held], fn, held ? VD_SMEM : 0, false);
    if (e != cudaSuccess) return (int) e;
    e = held ? launch_clusters(k_verify_draw<T, true>, A.n_seq, ctas, VD_THREADS, smem, A.n_drafts > 0, st, A) : launch_clusters(k_verify_draw<T, false>, A.n_seq, ctas, VD_THREADS, 0, A.n_drafts > 0, st, A);
    if (e == cudaSuccess) g_launches++;
    return (int) e;
}

}  // namespace
}  // namespace pb

using namespace pb;

namespace {
constexpr int VERIFY_CHUNKS = 64;      // of a row, at most
// rows over enough CTAs to fill the GPU, each with a batch of loads at least
int chunks_of(int64_t rows, int vocab, int elem) {
    const int64_t least = (int64_t) VR_ONCE * VR_THREADS * 16 / elem, most = (vocab + least - 1) / least, want = (16 * sm_count() + rows - 1) / rows;
    const int64_t n = want < most ? want : most;
    return (int) (n < 1 ? 1 : n > VERIFY_CHUNKS ? VERIFY_CHUNKS : n);
}
}  // namespace

extern "C" {

size_t pb200_verify_drafts_workspace_bytes(int64_t n_drafts) { return n_drafts >= 0 && n_drafts <= INT32_MAX ? (size_t) n_drafts * 2 * VERIFY_CHUNKS * sizeof(float4) + 16 : 0; }

int pb200_verify_drafts(int type, const void * target, int64_t ld_target, const void * draft, int64_t ld_draft, int n_vocab, int n_seq, const int32_t * start, int64_t n_drafts,
                        const int32_t * tokens, const float * inv_temp, const float * u_accept, const float * u_draw, int32_t * n_accepted, int32_t * out, int64_t ld_out, const int32_t * kv_len,
                        int32_t * kv_len_out, void * ws, size_t ws_bytes, void * stream) {
    const int eb = type == PB200_TYPE_F32 ? 4 : type == PB200_TYPE_F16 || type == PB200_TYPE_BF16 ? 2 : 0;
    if (!eb || n_vocab <= 0 || n_seq < 0 || n_drafts < 0 || n_drafts > INT32_MAX) return PB200_EINVAL;
    if (!target || ((uintptr_t) target & (eb - 1)) || ld_target < n_vocab || (draft && (((uintptr_t) draft & (eb - 1)) || ld_draft < n_vocab))) return PB200_EINVAL;
    if (!start || !u_draw || !n_accepted || !out || ld_out <= 0 || (kv_len == nullptr) != (kv_len_out == nullptr)) return PB200_EINVAL;
    if (n_drafts > 0 && (!tokens || !u_accept || !ws || ((uintptr_t) ws & 15) || ws_bytes < pb200_verify_drafts_workspace_bytes(n_drafts))) return PB200_EINVAL;
    if (n_vocab > 1 << 30 || n_seq > INT32_MAX / 8 || n_drafts * 2 > INT32_MAX / VERIFY_CHUNKS) return PB200_ENOTSUP;      // indices of the grids
    if (n_seq == 0) return 0;
    const Verify a{target, draft, ld_target, ld_draft, n_vocab, n_seq, start, n_drafts, tokens, inv_temp, u_accept, u_draw, n_accepted, out, ld_out, kv_len, kv_len_out, (float4 *) ws,
                   n_drafts > 0 ? chunks_of(n_drafts * (draft ? 2 : 1), n_vocab, eb) : 1};
    const cudaStream_t st = (cudaStream_t) stream;
    return type == PB200_TYPE_F32 ? verify_launch<float>(a, st) : type == PB200_TYPE_F16 ? verify_launch<__half>(a, st) : verify_launch<__nv_bfloat16>(a, st);
}

}  // extern "C"
