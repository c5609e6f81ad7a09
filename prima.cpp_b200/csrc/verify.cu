// prima.cpp_b200/csrc/verify.cu — verification of drafted tokens: how many of a sequence's drafts the target accepts, and the token that follows them.
//
// Mathematics.  With p and q the softmax of the target's and the draft's logits times t = 1 / temperature, drafted token x is accepted where u q(x) < p(x).  Behind the accepted ones comes a
// token from max(p - q, 0) at the place of the rejection, from p behind the last draft: by the inverse of the cumulative sum at v times the whole.  What is emitted then has the target's
// distribution, whatever the draft's.
//   rows    a CTA has a chunk of a row: its largest logit m and the sum of 2^((l - m) t log2 e), in 32 bits: a decision u q < p may change
//           where they are within 1e-5 of each other (additions one behind the other, up to 60 of a thread's, and exponents that are rounded three times; 1e-6 as a rule)
//   draw    a cluster has a sequence.  It joins its rows' chunks, decides, and adds up the weights that the token is drawn with, of one row, or of two with draft logits.  Weights and sums are in
//           64 bits: a cumulative sum of 100 000 weights with errors of 1e-8 each would give another token once in a thousand draws.  Each warp has the sum of a contiguous part; that in which the
//           token lies goes to all warps of its CTA once more, and a part of that is scanned.
//
// Bound.  rows: memory where there are many.  draw: no pipe is full (64 sequences: fp64 35 %, issue slots 39 %, 36 % of the warps): chains of loads and 64-bit instructions (a weight is a root of 16 from a
// table and a polynomial of degree 5), twice over two rows, and, for few sequences, of launch, row sums, cluster barriers and parts.  us: 64 sequences, 3.6 drafts each on the average, rows of 128 256
// in 32 bits, 117 (47 of them the rows, 5 TB/s); 24 with drafts from elsewhere, 151 937 in bf16, 33; one sequence, 3 drafts, 32 000, 17 to 19.  exp in 64 bits instead of the table 248, 69 and 23.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cfloat>
#include <climits>
#include <type_traits>

#include "../../include/prima_b200.h"
#include "cluster.cuh"
#include "launch.h"

extern std::atomic<uint64_t> g_launches;

namespace pb {
namespace {

constexpr int VERIFY_CHUNKS = 64;      // of a row, at most
constexpr int VR_THREADS = 256, VR_CTAS = 4, VR_ONCE = 4;      // rows: CTAs of an SM; vectors of 16 bytes to a thread at a time

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
__device__ __forceinline__ float raw(const float * p) { return *p; }
__device__ __forceinline__ float raw(const __half * p) { return __half2float(*p); }
__device__ __forceinline__ float raw(const __nv_bfloat16 * p) { return __bfloat162float(*p); }
template <typename T> __device__ __forceinline__ float get(const T * p) { return number(raw(p)); }
template <typename T> constexpr int vec() { return 16 / (int) sizeof(T); }
// vector v of a row of n: entries v * vec - skew and on, those outside -inf.  skew: entries between a 16-byte boundary and the row's first
template <typename T>
__device__ __forceinline__ void get_vec(const T * row, int n, int skew, int v, uint4 & w) {
    const int at = v * vec<T>() - skew;
    if (at >= 0 && at + vec<T>() <= n) w = __ldg(reinterpret_cast<const uint4 *>(row + at));
    else {
        T * e = reinterpret_cast<T *>(&w);
#pragma unroll
        for (int i = 0; i < vec<T>(); i++) e[i] = at + i >= 0 && at + i < n ? row[at + i] : T(-INFINITY);
    }
}
template <typename T> __device__ __forceinline__ int skew_of(const T * row) { return (int) (((uintptr_t) row & 15) / sizeof(T)); }

__device__ __forceinline__ float inv_temp_of(const Verify & A, int s) { return A.inv_temp ? A.inv_temp[s] : 1.f; }      // none where it is below 0 or no number

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
// weight of a logit relative to one that is larger, by half their difference (the whole one may be more than the largest number); c: of such a half to the power of two
__device__ __forceinline__ float weight(float l, float top, float c) { return ex2(fmaf(l, 0.5f, -0.5f * top) * c); }
// of 1 / temperature 0 the smallest number, so that times -inf it is no NaN; above 1e38 the largest, which leaves nothing of logits that are 1e-36 apart
__device__ __forceinline__ float half_to_power(float t) { return t == 0.f ? 1.4e-45f : fminf(t * 2.8853900817779268f, FLT_MAX); }
// sums of weights relative to the largest logit
struct Sum {
    float m = -INFINITY, l = 0.f;
    __device__ __forceinline__ void add(float m2, float l2, float c) {
        const float top = fmaxf(m, m2);
        if (top == INFINITY) l = (m == INFINITY ? l : 0.f) + (m2 == INFINITY ? l2 : 0.f);
        else if (top > -INFINITY) l = l * weight(m, top, c) + l2 * weight(m2, top, c);
        m = top;
    }
};

template <typename T>
__global__ void __launch_bounds__(VR_THREADS, VR_CTAS) k_verify_rows(const __grid_constant__ Verify A) {
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
    const float t = inv_temp_of(A, s), c = half_to_power(t);
    Sum sum;
    int arg = INT_MAX;
    const bool greedy = t == INFINITY;
    auto take = [&](auto once, int v0, const uint4 * w) {   // so many vectors from v0 on
        constexpr int ONCE = decltype(once)::value;
        float top = -INFINITY;
        auto entry = [&](int k, int e) { return number(raw(reinterpret_cast<const T *>(&w[k]) + e)); };
#pragma unroll
        for (int k = 0; k < ONCE; k++)
#pragma unroll
            for (int e = 0; e < VEC; e++) top = fmaxf(top, entry(k, e));
        if (greedy) {
            if (top > sum.m) {
                sum.m = top;
#pragma unroll
                for (int k = ONCE - 1; k >= 0; k--)
#pragma unroll
                    for (int e = VEC - 1; e >= 0; e--)
                        if (entry(k, e) == top) arg = (v0 + k * VR_THREADS) * VEC - skew + e;
            }
        } else if (top > -INFINITY) {
            float l = 0.f;
            if (top == INFINITY) {
#pragma unroll
                for (int k = 0; k < ONCE; k++)
#pragma unroll
                    for (int e = 0; e < VEC; e++) l += entry(k, e) == INFINITY ? 1.f : 0.f;
            } else {
#pragma unroll
                for (int k = 0; k < ONCE; k++)
#pragma unroll
                    for (int e = 0; e < VEC; e++) l += weight(entry(k, e), top, c);
            }
            sum.add(top, l, c);
        }
    };
    // whole batches, the next one on its way beside the one at hand
    const int batch = VR_ONCE * VR_THREADS;
    int v0 = from + tid, whole = (to - from) / batch;
    uint4 now[VR_ONCE];
    auto ask = [&](int v, uint4 (&w)[VR_ONCE]) {
#pragma unroll
        for (int k = 0; k < VR_ONCE; k++) get_vec(src, A.vocab, skew, v + k * VR_THREADS, w[k]);
    };
    if (whole > 0) ask(v0, now);
    for (; whole > 0; whole--, v0 += batch) {
        uint4 next[VR_ONCE];
        if (whole > 1) ask(v0 + batch, next);
        take(std::integral_constant<int, VR_ONCE>(), v0, now);
#pragma unroll
        for (int k = 0; k < VR_ONCE; k++) now[k] = next[k];
    }
    for (; v0 < to; v0 += VR_THREADS) {
        get_vec(src, A.vocab, skew, v0, now[0]);
        take(std::integral_constant<int, 1>(), v0, now);
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

// 2^(y / 16) in 64 bits for y from -16 * 1000 to 0: the whole part of y goes to the exponent and to one of 16 roots, 2^(r / 16) of the rest (up to a half) is the polynomial that agrees
// with it at the six Chebyshev nodes: within 2^-47 of it.  (Without roots nine products instead of five: 64 sequences of 128 256 logits 4 us more.)
__device__ __forceinline__ double power_of_two(double y, const double * roots) {
    constexpr double ROUND = 6755399441055744.0;          // 1.5 * 2^52: a sum with it has the whole number in its last bits
    const double z = y + ROUND, r = y - (z - ROUND);
    const int k = __double2loint(z);
    double p = 1.2716085030349987e-09;
    p = fma(p, r, 1.467644462189871e-07);
    p = fma(p, r, 1.355080777749983e-05);
    p = fma(p, r, 0.000938384792486206);
    p = fma(p, r, 0.04332169878499661);
    p = fma(p, r, 1.0000000000000044) * roots[k & 15];
    return __hiloint2double(__double2hiint(p) + ((k & ~15) << 16), __double2loint(p));
}
// The weights of a row's logits, the largest of them m; none is taken for less than 2^-1000, masked entries and what is no number among them: NOTHING is less than that, and a sum of them.
// The difference comes first, in 64 bits, then the temperature, then the floor: a floor under the logits themselves would be off by half a step of m times 1 / temperature, which has no bound.
// The floor by the high word, as a whole number (y is 0 or less, and -inf above all others): 64 sequences of 128 256 logits 117 us, by a comparison of 64-bit numbers 121
constexpr double NOTHING = 1e-290, FLOOR = -16000.0;
constexpr uint32_t FLOOR_HIGH = 0xc0cf4000u;       // the high word of FLOOR, whose low one is 0
struct Weights {
    double c, m;               // c: never 0: times -inf it is no NaN
    bool step;                 // a largest logit of +inf: the same weight for all of these, none for others
    const double * roots;      // 2^(i / 16)
    __device__ __forceinline__ Weights(float m, float t, const double * roots) : c(fmax((double) t * (16 * 1.4426950408889634), 1e-300)), m(m), step(m == INFINITY), roots(roots) {}
    template <int N> __device__ __forceinline__ void operator()(const float (&l)[N], double (&w)[N]) const {
        if (step) {
#pragma unroll
            for (int i = 0; i < N; i++) w[i] = l[i] == INFINITY ? 1.0 : 0.0;
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) {
                const double y = ((double) number(l[i]) - m) * c;
                w[i] = power_of_two((uint32_t) __double2hiint(y) <= FLOOR_HIGH ? y : FLOOR, roots);
            }
        }
    }
    __device__ __forceinline__ double operator()(float l) const {
        const float x[1] = {l};
        double w[1];
        (*this)(x, w);
        return w[0];
    }
};

template <int WARPS> struct VdSmem {
    double warp[WARPS][2], roots[16];
    double z[2], all[2];       // what the other CTAs read: sums of either row, of the weights
    float top;
    int arg, first;
};

// sum of the warp's numbers in the lanes' order, of the first parts: `front` and the lanes up to the one that ends beyond x (where rounding leaves none, the last that has any) -> that lane
__device__ __forceinline__ int find(double w, double x, double & front) {
    const int lane = threadIdx.x & 31;
    double upto = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
    }
    const uint32_t some = __ballot_sync(0xffffffffu, w > NOTHING), above = __ballot_sync(0xffffffffu, w > NOTHING && front + upto > x);
    const int at = above ? __ffs((int) above) - 1 : some ? 31 - __clz((int) some) : 0;
    front += __shfl_sync(0xffffffffu, upto - w, at);
    return at;
}

// a row's chunks, two to a lane of a warp
struct Chunks {
    float4 p[VERIFY_CHUNKS / 32];
    __device__ __forceinline__ Chunks(const float4 * parts, int chunks) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int k = 0; k < VERIFY_CHUNKS / 32; k++) p[k] = lane + 32 * k < chunks ? __ldcg(&parts[lane + 32 * k]) : make_float4(-INFINITY, 0.f, __int_as_float(INT_MAX), 0.f);
    }
    __device__ __forceinline__ float top() const {
        float m = -INFINITY;
#pragma unroll
        for (int k = 0; k < VERIFY_CHUNKS / 32; k++) m = fmaxf(m, p[k].x);
        return warp_max(m);
    }
    __device__ __forceinline__ int first(float m) const {           // of the largest
        int arg = INT_MAX;
#pragma unroll
        for (int k = 0; k < VERIFY_CHUNKS / 32; k++)
            if (p[k].x == m) arg = min(arg, __float_as_int(p[k].z));
        return __reduce_min_sync(0xffffffffu, arg);
    }
    __device__ __forceinline__ double chance(int x, float lx, float t, const double * roots) const {   // p(x)
        const float m = top();
        if (m == -INFINITY || !(t >= 0.f)) return 0.0;
        if (t == INFINITY) return first(m) == x ? 1.0 : 0.0;
        const Weights w(m, t, roots);
        double l = 0.0;
#pragma unroll
        for (int k = 0; k < VERIFY_CHUNKS / 32; k++)
            if (p[k].x > -INFINITY) l += p[k].y * w(p[k].x);
        l = warp_sum_d(l);
        const double of_x = w(lx);
        return of_x > NOTHING ? of_x / l : 0.0;
    }
};

template <typename T, int WARPS>
__global__ void __launch_bounds__(32 * WARPS, 32 / WARPS) k_verify_draw(const __grid_constant__ Verify A) {
    constexpr int THREADS = 32 * WARPS;
    __shared__ VdSmem<WARPS> S;
    const uint32_t rank = cluster_rank(), ctas = cluster_size();
    const int s = blockIdx.x / ctas, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t a = A.start[s], b = A.start[s + 1];
    const bool good = a >= 0 && b >= a && b <= A.n_drafts;
    const int drafts = good ? (int) (b - a) : 0;
    const float t = inv_temp_of(A, s);
    if (tid == 0) S.first = drafts;
    if (tid < 16) S.roots[tid] = exp2(tid * 0.0625);
    // this warp's first draft: what is known of it ahead of the rows' sums
    int token = -1;
    float of_p = -INFINITY, of_q = -INFINITY, u = 0.f;
    auto ask = [&](int i) {
        token = A.tokens[a + i];
        u = A.u[a + i];
        if (token < 0 || token >= A.vocab) return;
        of_p = get((const T *) A.target + (a + i + s) * A.ld_target + token);
        if (A.draft) of_q = get((const T *) A.draft + (a + i) * A.ld_draft + token);
    };
    if (warp < drafts) ask(warp);
    __syncthreads();
    pdl_wait();                                             // the rows' sums
    if (!good) return;                                      // (all CTAs of the cluster)
    for (int i = warp; i < drafts; i += WARPS) {
        if (i != warp) ask(i);
        bool ok = false;
        if (token >= 0 && token < A.vocab) {
            const Chunks p(A.parts + (a + i) * A.chunks, A.chunks), q(A.parts + (A.draft ? A.n_drafts + a + i : a + i) * A.chunks, A.chunks);
            ok = (double) u * (A.draft ? q.chance(token, of_q, t, S.roots) : 1.0) < p.chance(token, of_p, t, S.roots);
        }
        if (!ok && lane == 0) atomicMin(&S.first, i);
    }
    __syncthreads();
    const int acc = S.first;
    const bool rejected = acc < drafts;
    const int out_of = rejected && !A.draft ? A.tokens[a + acc] : -1;       // a token whose weight is 0
    const T * const row_p = (const T *) A.target + (a + s + acc) * A.ld_target, * const row_q = rejected && A.draft ? (const T *) A.draft + (a + acc) * A.ld_draft : nullptr;
    if (rank == 0) {
        for (int64_t i = tid; i < acc && i < A.ld_out; i += THREADS) A.out[s * A.ld_out + i] = A.tokens[a + i];
        if (tid == 0) {
            A.accepted[s] = acc;
            if (A.kv_len) A.kv_len_out[s] = A.kv_len[s] - (drafts - acc);
        }
    }
    // this CTA's part of the vocabulary, and this warp's, both even to a load of a warp
    const int loads = (A.vocab + 31) / 32, l0 = (int) ((int64_t) loads * rank / ctas), l1 = (int) ((int64_t) loads * (rank + 1) / ctas);
    const int from = 32 * (l0 + (int) ((int64_t) (l1 - l0) * warp / WARPS)), to = min(A.vocab, 32 * (l0 + (int) ((int64_t) (l1 - l0) * (warp + 1) / WARPS)));

    // ---- the rows' largest logits: of those that were looked at, from their chunks ----
    float m[2] = {-INFINITY, -INFINITY};
    int arg = INT_MAX;
    if (rejected) {
        const Chunks p(A.parts + (a + acc) * A.chunks, A.chunks), q(A.parts + (row_q ? A.n_drafts + a + acc : a + acc) * A.chunks, A.chunks);
        m[0] = p.top();
        m[1] = q.top();
        arg = p.first(m[0]);
    } else {
        constexpr int ONCE = 8;
        for (int i0 = from + lane; i0 < to; i0 += 32 * ONCE) {
            float x[ONCE];
#pragma unroll
            for (int k = 0; k < ONCE; k++) x[k] = i0 + 32 * k < to ? raw(row_p + i0 + 32 * k) : -INFINITY;
#pragma unroll
            for (int k = 0; k < ONCE; k++)
                if (x[k] > m[0]) { m[0] = x[k]; arg = i0 + 32 * k; }
        }
        const float own = m[0];
        m[0] = warp_max(m[0]);
        arg = __reduce_min_sync(0xffffffffu, own == m[0] && own > -INFINITY ? arg : INT_MAX);
        if (lane == 0) { S.warp[warp][0] = m[0]; S.warp[warp][1] = arg; }
        __syncthreads();
        const float top = lane < WARPS ? (float) S.warp[lane % WARPS][0] : -INFINITY, most = warp_max(top);
        const int first = __reduce_min_sync(0xffffffffu, top == most && lane < WARPS ? (int) S.warp[lane % WARPS][1] : INT_MAX);
        if (tid == 0) { S.top = most; S.arg = first; }
        cluster_sync();
        const float far = lane < ctas ? remote(&S.top, lane % ctas) : -INFINITY;
        m[0] = warp_max(far);
        arg = __reduce_min_sync(0xffffffffu, far == m[0] && lane < ctas ? remote(&S.arg, lane % ctas) : INT_MAX);
    }
    if (m[0] == -INFINITY || !(t >= 0.f) || t == INFINITY) {       // no weights; all of it on one
        if (rank == 0 && tid == 0 && acc < A.ld_out) A.out[s * A.ld_out + acc] = t == INFINITY && m[0] > -INFINITY ? arg : -1;
        cluster_sync();                                     // (others read this CTA's numbers)
        return;
    }

    // ---- weights ----
    const Weights wp(m[0], t, S.roots), wq(m[1], t, S.roots);
    const bool minus_q = row_q && m[1] > -INFINITY;         // (a draft row without a number takes nothing away)
    constexpr int ONCE = 4;
    // f(first entry, logits of p, of q) for the entries i0 .. i1 - 1, ONCE of a lane at a time, 32 entries from each other; those outside are -inf
    auto walk = [&](int i0, int i1, auto && f) {
        for (i0 += lane; i0 < i1; i0 += 32 * ONCE) {
            float lp[ONCE], lq[ONCE];
#pragma unroll
            for (int k = 0; k < ONCE; k++) {
                lp[k] = i0 + 32 * k < i1 ? raw(row_p + i0 + 32 * k) : -INFINITY;
                lq[k] = minus_q && i0 + 32 * k < i1 ? raw(row_q + i0 + 32 * k) : -INFINITY;
            }
            f(i0, lp, lq);
        }
    };
    auto add_up = [&](const double (&w)[ONCE]) {
        double x = w[0];
#pragma unroll
        for (int k = 1; k < ONCE; k++) x += w[k];
        return x;
    };
    double part_p = 0.0, part_q = 0.0;                      // of a weight its part of the row's
    if (minus_q) {
        double x = 0.0, y = 0.0;
        walk(from, to, [&](int, const float (&lp)[ONCE], const float (&lq)[ONCE]) {
            double p[ONCE], q[ONCE];
            wp(lp, p);
            wq(lq, q);
            x += add_up(p);
            y += add_up(q);
        });
        x = warp_sum_d(x);
        y = warp_sum_d(y);
        if (lane == 0) { S.warp[warp][0] = x; S.warp[warp][1] = y; }
        __syncthreads();
        if (warp == 0) {
            x = warp_sum_d(lane < WARPS ? S.warp[lane % WARPS][0] : 0.0);
            y = warp_sum_d(lane < WARPS ? S.warp[lane % WARPS][1] : 0.0);
            if (lane == 0) { S.z[0] = x; S.z[1] = y; }
        }
        cluster_sync();
        part_p = 1.0 / warp_sum_d(lane < ctas ? remote(&S.z[0], lane % ctas) : 0.0);
        part_q = 1.0 / warp_sum_d(lane < ctas ? remote(&S.z[1], lane % ctas) : 0.0);
    }
    bool rest = minus_q || out_of >= 0;                     // max(p - q, 0), or p
    auto weights = [&](int i0, int step, const float (&lp)[ONCE], const float (&lq)[ONCE], double (&w)[ONCE]) {
        wp(lp, w);
        if (rest && minus_q) {
            double q[ONCE];
            wq(lq, q);
#pragma unroll
            for (int k = 0; k < ONCE; k++) w[k] = fmax(__dmul_rn(w[k], part_p) - __dmul_rn(q[k], part_q), 0.0);      // either rounded by itself: of equal rows nothing is left
        } else if (rest)
#pragma unroll
            for (int k = 0; k < ONCE; k++) w[k] = i0 + step * k == out_of ? 0.0 : w[k];
    };
    // The warps' sums; the CTA and the warp in whose entries the token is; that warp's entries, in as many pieces, once more; the piece
    double x = 0.0, front = 0.0;
    int lo = from, hi = to, w0 = 0, w1 = 0, piece = 0;
    for (int round = 0;; round++) {
        double mine = 0.0;
        walk(lo, hi, [&](int at, const float (&lp)[ONCE], const float (&lq)[ONCE]) {
            double w[ONCE];
            weights(at, 32, lp, lq, w);
            mine += add_up(w);
        });
        mine = warp_sum_d(mine);
        __syncthreads();
        if (lane == 0) S.warp[warp][0] = mine;
        __syncthreads();
        mine = lane < WARPS ? S.warp[lane % WARPS][0] : 0.0;
        if (piece > 0) {
            lo = w0 + piece * find(mine, x, front);
            hi = min(w1, lo + piece);
            break;
        }
        const double all = warp_sum_d(mine);
        if (tid == 0) S.all[round] = all;
        cluster_sync();
        const double far = lane < ctas ? remote(&S.all[round], lane % ctas) : 0.0, total = warp_sum_d(far);
        if (!(total > NOTHING) && rest) {                   // nothing is left: from p
            rest = false;
            continue;
        }
        x = (double) A.v[s] * total;
        const int owner = find(far, x, front);
        cluster_sync();                                     // nobody reads this CTA's numbers from here on
        if (owner != (int) rank) return;
        const int w = find(mine, x, front);
        w0 = 32 * (l0 + (int) ((int64_t) (l1 - l0) * w / WARPS));
        w1 = min(A.vocab, 32 * (l0 + (int) ((int64_t) (l1 - l0) * (w + 1) / WARPS)));
        piece = ((w1 - w0 + WARPS - 1) / WARPS + 31) & ~31;
        lo = w0 + warp * piece;
        hi = min(w1, lo + piece);
    }
    if (warp != 0) return;
    // an even part of them to each lane, until a part is one entry
    while (hi - lo > 1) {
        const int each = (hi - lo + 31) / 32, i0 = min(hi, lo + lane * each), i1 = min(hi, i0 + each);
        double own = 0.0;
        for (int i = i0; i < i1; i += ONCE) {
            float lp[ONCE], lq[ONCE];
            double some[ONCE];
#pragma unroll
            for (int k = 0; k < ONCE; k++) {
                lp[k] = i + k < i1 ? raw(row_p + i + k) : -INFINITY;
                lq[k] = i + k < i1 && minus_q ? raw(row_q + i + k) : -INFINITY;
            }
            weights(i, 1, lp, lq, some);
            own += add_up(some);
        }
        const int at = find(own, x, front);
        lo += at * each;
        hi = min(hi, lo + each);
    }
    if (lane == 0 && acc < A.ld_out) A.out[s * A.ld_out + acc] = lo;
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
    const int ctas = A.vocab > 16384 ? 8 : A.vocab > 8192 ? 4 : A.vocab > 4096 ? 2 : 1;
    const int64_t warps = 32 * sm_count() / ((int64_t) A.n_seq * ctas);
    const bool after = A.n_drafts > 0;
    const cudaError_t e = warps >= 16 ? launch_clusters(k_verify_draw<T, 16>, A.n_seq, ctas, 512, 0, after, st, A)
                                      : launch_clusters(k_verify_draw<T, 8>, A.n_seq, ctas, 256, 0, after, st, A);
    if (e == cudaSuccess) g_launches++;
    return (int) e;
}

}  // namespace
}  // namespace pb

using namespace pb;

namespace {
// Chunks of a row: as many CTAs as the GPU runs at once take a round; that number of chunks whose rounds of whole batches of loads, and a batch's time for each CTA's start and end, are fewest
int chunks_of(int64_t rows, int vocab, int elem) {
    const int64_t batch = (int64_t) VR_ONCE * VR_THREADS * 16 / elem, batches = (vocab + batch - 1) / batch, at_once = VR_CTAS * sm_count();
    int64_t best = 1, cost = INT64_MAX;
    for (int64_t n = 1; n <= VERIFY_CHUNKS && n <= batches; n++) {
        const int64_t k = (rows * n + at_once - 1) / at_once * ((batches + n - 1) / n + 1);
        if (k < cost) { cost = k; best = n; }
    }
    return (int) best;
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
