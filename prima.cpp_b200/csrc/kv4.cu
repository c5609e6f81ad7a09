// prima.cpp_b200/csrc/kv4.cu — what writes and moves the cells of the 4-bit cache (kv4.cuh): rows of a step into their cells with the norms of queries and
// keys and the rotation on the way, their values back, pages of a fork, cells that are kept.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "../../include/prima_b200.h"
#include "kv4.cuh"

namespace pb {
namespace {

constexpr int KA_THREADS = 256, KA_WARPS = KA_THREADS / 32, KA_MANY = 2;

template <typename T>
struct AppendParams {
    Kv4 cache;
    const T * q; const T * k; const T * v; T * q_out;
    int64_t ldq, ldqo, ldk, ldv;
    int n_head, n_tokens;
    const int64_t * cells; const int32_t * pos;
    const float * q_norm; const float * k_norm;
    float eps;
};
__device__ __forceinline__ void raw4(const float * p, uint32_t (&w)[4]) { *reinterpret_cast<uint4 *>(w) = *reinterpret_cast<const uint4 *>(p); }
template <typename T> __device__ __forceinline__ void raw4(const T * p, uint32_t (&w)[2]) { *reinterpret_cast<uint2 *>(w) = *reinterpret_cast<const uint2 *>(p); }

// the sum of four squares to 47 bits: products and sums of 32 bits with what their roundings left (two conversions to 64 bits where four numbers are eight operations); exact: squares of
// numbers of T have 24 bits at most.  (The larger and the smaller of a NaN are no NaN: the sum has it.)
template <typename T>
__device__ __forceinline__ double squares(const float (&x)[4]) {
    constexpr bool exact = sizeof(T) == 2;
    float hi = __fmul_rn(x[0], x[0]), lo = exact ? 0.f : fmaf(x[0], x[0], -hi);
#pragma unroll
    for (int i = 1; i < 4; i++) {
        const float p = __fmul_rn(x[i], x[i]), big = fmaxf(hi, p), small = fminf(hi, p), s = __fadd_rn(hi, p), left = __fsub_rn(small, __fsub_rn(s, big));
        lo += exact ? left : left + fmaf(x[i], x[i], -p);
        hi = s;
    }
    if (!(hi > 1e-30f && hi < 1e38f)) {   // squares that leave the range of 32 bits
        double sum = 0.0;
        for (float v : x) sum += (double) v * (double) v;
        return sum;
    }
    return (double) hi + (double) lo;
}
// 1 / sqrt(v) rounded to 32 bits: two steps of Newton's method in 64 bits from the 32-bit function (a square root and a division of 64 bits take five times as long)
__device__ __forceinline__ float inverse_root(double v) {
    if (!(v > 1e-30 && v < 1e38)) return (float) (1.0 / sqrt(v));
    double y = (double) rsqrtf((float) v);
    y = y * (1.5 - 0.5 * v * y * y);
    y = y * (1.5 - 0.5 * v * y * y);
    return (float) y;
}

// Bound: instructions: a row's norm and rotation, and a stored row's scale and steps, about as much again each as reading and writing a row of queries.  us, 2048 tokens of 32 heads over 8
// of 128, bf16: 22 (and 6 for k_kv4_load; floor 8.4 of both); 64 tokens in F32 3.  A head to a warp and angles once for 8 rows 57; roots and quotients of 64 and 32 bits 42; four tokens to
// a CTA (some SMs have four of these, others three), and steps by conversions, 28.
// A CTA takes TOKENS tokens at a time and a part of their heads, a warp R heads of q, of k or of v at a time (R rows on their way together): D / 4 lanes hold a row, four neighbouring numbers
// each.  What decides which of 16 steps a number falls to is computed so that it does not depend on an order: the mean of squares and the angles in 64 bits, rounded
// once, products and sums of the rotation in 32 bits without contraction.
template <typename T, int D, int TOKENS, int R>
__global__ void __launch_bounds__(KA_THREADS, 4) k_kv4_append(const __grid_constant__ AppendParams<T> P, const __grid_constant__ Kv4Rope RP) {
    constexpr int LPR = D / 4, RPW = 32 / LPR, HEADS = R * RPW;      // lanes to a row, rows to a warp's instruction, heads to an item
    __shared__ float2 cs[TOKENS][D / 2];
    const int lane = threadIdx.x & 31;
    const int pairs = RP.n_dims / 2, hk = P.cache.n_head_kv;
    const int sub = lane / LPR, l = lane % LPR, d = 4 * l, b = d / 32;
    const int of_q = (P.n_head + HEADS - 1) / HEADS, of_kv = (hk + HEADS - 1) / HEADS, of_token = of_q + 2 * of_kv;
    const int step = KA_WARPS * gridDim.y;
    uint32_t raw[R][sizeof(T) == 4 ? 4 : 2];
    const int t0 = blockIdx.x * TOKENS;
    int t = 0, kind = 0, head0 = 0, heads = 0;   // of the item at hand: token, 0 q 1 k 2 v, its first head, heads there are
    auto ask = [&](int item) {
        t = item / of_token;
        const int i = item - t * of_token;
        kind = i < of_q ? 0 : i < of_q + of_kv ? 1 : 2;
        head0 = (kind == 0 ? i : kind == 1 ? i - of_q : i - of_q - of_kv) * HEADS;
        heads = kind == 0 ? P.n_head : hk;
        const int64_t row = t0 + t;
        const T * src = (kind == 0 ? P.q + row * P.ldq : kind == 1 ? P.k + row * P.ldk : P.v + row * P.ldv) + d;
#pragma unroll
        for (int r = 0; r < R; r++) {
            const int head = head0 + r * RPW + sub;
            if (head < heads) raw4(src + (int64_t) head * D, raw[r]);
            else
                for (uint32_t & w : raw[r]) w = 0u;
        }
    };
    const int tokens = min(TOKENS, P.n_tokens - t0), items = tokens * of_token;
    int item = blockIdx.y * KA_WARPS + (threadIdx.x >> 5);
    if (item < items) ask(item);                                     // on its way beside the angles
    for (int i = threadIdx.x; i < tokens * pairs; i += KA_THREADS) {
        const int at = i / pairs, pair = i - at * pairs;
        const double a = (double) P.pos[t0 + at] * RP.w[pair] / (RP.freq_factors ? (double) RP.freq_factors[pair] : 1.0);
        double s, c;
        sincos(a, &s, &c);
        cs[at][pair] = make_float2(__fmul_rn((float) c, RP.mscale), __fmul_rn((float) s, RP.mscale));
    }
    __syncthreads();
    for (; item < items; item += step) {
        float x[R][4];
#pragma unroll
        for (int r = 0; r < R; r++) {
            const float4 v = load4(reinterpret_cast<const T *>(raw[r]));
            x[r][0] = v.x; x[r][1] = v.y; x[r][2] = v.z; x[r][3] = v.w;
        }
        const int at = t, is = kind, first = head0, n = heads;
        if (item + step < items) ask(item + step);
        const float * w = is == 0 ? P.q_norm : is == 1 ? P.k_norm : nullptr;
        if (w) {
            const float4 w4 = load4(w + d);
            float f[R];
            if constexpr (R == 4) {   // four rows at once: each step of the sum halves the rows that a lane adds up for, until a quarter of a row's lanes has one
                constexpr int H = LPR / 2, Q = LPR / 4;
                double v[4];
#pragma unroll
                for (int r = 0; r < 4; r++) v[r] = squares<T>(x[r]);
                const bool h = lane & H, q = lane & Q;
#pragma unroll
                for (int r = 0; r < 2; r++) v[r] = (h ? v[r + 2] : v[r]) + __shfl_xor_sync(0xffffffffu, h ? v[r] : v[r + 2], H);
                double sum = (q ? v[1] : v[0]) + __shfl_xor_sync(0xffffffffu, q ? v[0] : v[1], Q);
#pragma unroll
                for (int o = Q / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                const float mine = inverse_root(sum * (1.0 / D) + (double) P.eps);
#pragma unroll
                for (int r = 0; r < 4; r++) f[r] = __shfl_sync(0xffffffffu, mine, sub * LPR + (r >> 1) * H + (r & 1) * Q);
            } else {
#pragma unroll
                for (int r = 0; r < R; r++) {
                    double sum = squares<T>(x[r]);
#pragma unroll
                    for (int o = LPR / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                    f[r] = inverse_root(sum * (1.0 / D) + (double) P.eps);
                }
            }
#pragma unroll
            for (int r = 0; r < R; r++) {
                x[r][0] = __fmul_rn(__fmul_rn(x[r][0], f[r]), w4.x);
                x[r][1] = __fmul_rn(__fmul_rn(x[r][1], f[r]), w4.y);
                x[r][2] = __fmul_rn(__fmul_rn(x[r][2], f[r]), w4.z);
                x[r][3] = __fmul_rn(__fmul_rn(x[r][3], f[r]), w4.w);
            }
        }
        if (is < 2 && pairs > 0) {
            const bool turns = d < 2 * pairs;
            if (RP.mode == 0) {                                      // neighbours: both in this lane
                const float2 a0 = turns ? cs[at][d / 2] : make_float2(1.f, 0.f), a1 = turns ? cs[at][d / 2 + 1] : make_float2(1.f, 0.f);
                if (turns) {
#pragma unroll
                    for (int r = 0; r < R; r++) {
                        const float y0 = x[r][0], y1 = x[r][1], y2 = x[r][2], y3 = x[r][3];
                        x[r][0] = __fsub_rn(__fmul_rn(y0, a0.x), __fmul_rn(y1, a0.y));
                        x[r][1] = __fadd_rn(__fmul_rn(y0, a0.y), __fmul_rn(y1, a0.x));
                        x[r][2] = __fsub_rn(__fmul_rn(y2, a1.x), __fmul_rn(y3, a1.y));
                        x[r][3] = __fadd_rn(__fmul_rn(y2, a1.y), __fmul_rn(y3, a1.x));
                    }
                }
            } else {                                                 // halves: the other one pairs / 4 lanes away
                const bool lower = d < pairs;
                const int other = lower ? lane + pairs / 4 : lane - pairs / 4;
                float2 a[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    a[i] = turns ? cs[at][lower ? d + i : d + i - pairs] : make_float2(1.f, 0.f);
                    if (lower) a[i].y = -a[i].y;
                }
#pragma unroll
                for (int r = 0; r < R; r++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float y = __shfl_sync(0xffffffffu, x[r][i], other);
                        if (turns) x[r][i] = __fadd_rn(__fmul_rn(x[r][i], a[i].x), __fmul_rn(y, a[i].y));
                    }
            }
        }
        if (is == 0) {
            T * to = P.q_out + (t0 + at) * P.ldqo + d;
#pragma unroll
            for (int r = 0; r < R; r++) {
                const int head = first + r * RPW + sub;
                if (head < n) store4(to + (int64_t) head * D, make_float4(x[r][0], x[r][1], x[r][2], x[r][3]));
            }
            continue;
        }
        const int64_t cell = P.cells[t0 + at];
        if (cell < 0 || cell >= P.cache.n_pages * KV4_CELLS) continue;
        const int c = (int) (cell % KV4_CELLS);
        uint8_t * page = kv4_chunk<D>(P.cache, cell / KV4_CELLS, 0);
#pragma unroll
        for (int r = 0; r < R; r++) {
            // the block's number of largest magnitude (of several, the first), scale, bits
            float most = 0.f;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                x[r][i] = kv4_finite(x[r][i]);
                if (i == 0 || fabsf(x[r][i]) > fabsf(most)) most = x[r][i];
            }
            float top = fabsf(most);
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const uint32_t who = __ballot_sync(0xffffffffu, fabsf(most) == top) & (0xffu << (lane & 24));
            const float scale = kv4_scale_of(__shfl_sync(0xffffffffu, most, __ffs((int) who) - 1));
            uint32_t m[4];
            kv4_bits_of(x[r], scale, scale == 0.f ? 0.f : __frcp_rn(scale), m);
            const int head = first + r * RPW + sub;
            uint8_t * chunk = page + (int64_t) head * kv4_chunk_bytes(D);
            if (is == 1) {
                uint32_t word = (m[0] | m[1] << 16 | m[2] << 4 | m[3] << 20) << (8 * (l & 1));
                word |= __shfl_xor_sync(0xffffffffu, word, 1);
                if (head < n && (l & 1) == 0) *reinterpret_cast<uint32_t *>(chunk + kv4_k_word(D, c, (d / 8) % 4, b)) = word;
            } else if (head < n)
                *reinterpret_cast<uint16_t *>(chunk + kv4_rows_bytes(D) + kv4_v_word(D, c, (d / 4) % 8, b)) = (uint16_t) (m[0] | m[1] << 4 | m[2] << 8 | m[3] << 12);
            if (head < n && (l & 7) == 0)
                *reinterpret_cast<__half *>(chunk + 2 * kv4_rows_bytes(D) + (is == 2 ? kv4_scales_bytes(D) : 0) + kv4_scale(D, c, b)) = __float2half_rn(scale);
        }
    }
}

template <typename T, int D>
__global__ void __launch_bounds__(256) k_kv4_load(const Kv4 cache, const int64_t * cells, int64_t n, T * k, int64_t ldk, T * v, int64_t ldv) {
    constexpr int LPR = D / 4;
    const int64_t item = ((int64_t) blockIdx.x * 256 + threadIdx.x) / LPR;      // (cell, head)
    const int d = 4 * (threadIdx.x % LPR), b = d / 32;
    if (item >= n * cache.n_head_kv) return;
    const int64_t i = item / cache.n_head_kv, cell = cells[i];
    const int head = (int) (item % cache.n_head_kv);
    if (cell < 0 || cell >= cache.n_pages * KV4_CELLS) return;
    const int at = (int) (cell % KV4_CELLS);
    const uint8_t * chunk = kv4_chunk<D>(cache, cell / KV4_CELLS, head);
    const uint8_t * scales = chunk + 2 * kv4_rows_bytes(D) + kv4_scale(D, at, b);
    if (k) {
        const uint32_t w = *reinterpret_cast<const uint32_t *>(chunk + kv4_k_word(D, at, (d / 8) % 4, b)) >> (8 * ((d / 4) & 1));
        const float s = __half2float(*reinterpret_cast<const __half *>(scales));
        store4(k + i * ldk + (int64_t) head * D + d, make_float4((float) ((int) (w & 15) - 8) * s, (float) ((int) (w >> 16 & 15) - 8) * s, (float) ((int) (w >> 4 & 15) - 8) * s,
                                                                 (float) ((int) (w >> 20 & 15) - 8) * s));
    }
    if (v) {
        const uint32_t w = *reinterpret_cast<const uint16_t *>(chunk + kv4_rows_bytes(D) + kv4_v_word(D, at, (d / 4) % 8, b));
        const float s = __half2float(*reinterpret_cast<const __half *>(scales + kv4_scales_bytes(D)));
        store4(v + i * ldv + (int64_t) head * D + d, make_float4((float) ((int) (w & 15) - 8) * s, (float) ((int) (w >> 4 & 15) - 8) * s, (float) ((int) (w >> 8 & 15) - 8) * s,
                                                                 (float) ((int) (w >> 12) - 8) * s));
    }
}

// Bound: memory.  48 pages of 2.4 MB, three copies of each source: 27 us (151 MB read once and written; floor 23).  One 16-byte piece a thread on its way: 34.
constexpr int KC_PAIRS = 256, KC_ONCE = 4;
struct CopyPairs { int32_t src[KC_PAIRS], dst[KC_PAIRS]; };
__global__ void __launch_bounds__(256) k_kv4_copy_pages(uint8_t * pages, int64_t page_bytes, const __grid_constant__ CopyPairs p) {
    const uint4 * s = reinterpret_cast<const uint4 *>(pages + p.src[blockIdx.y] * page_bytes);
    uint4 * d = reinterpret_cast<uint4 *>(pages + p.dst[blockIdx.y] * page_bytes);
    const int64_t n = page_bytes / 16;
    for (int64_t i0 = (int64_t) blockIdx.x * (KC_ONCE * 256) + threadIdx.x; i0 < n; i0 += (int64_t) gridDim.x * (KC_ONCE * 256)) {
        uint4 v[KC_ONCE];
#pragma unroll
        for (int i = 0; i < KC_ONCE; i++)
            if (i0 + i * 256 < n) v[i] = s[i0 + i * 256];
#pragma unroll
        for (int i = 0; i < KC_ONCE; i++)
            if (i0 + i * 256 < n) d[i0 + i * 256] = v[i];
    }
}

// Eight threads to a cell: each an eighth of its key row, one of the eight words of its value row (which lie in another order there and here) and a scale or two.  What the tables
// say serves KM_CHUNKS chunks (heads and layers), which are on their way together.  Bound: memory, by pieces of 64 bytes: 4000 of 8000 cells, 64 chunks, 20.5 us (floor 11.3); two bytes of
// values at a time and a chunk to a thread 38.
constexpr int KM_CHUNKS = 8;
template <int D>
__global__ void __launch_bounds__(256) k_kv4_compact(uint8_t * pages, int64_t n_pages, int chunks, const int32_t * from, int64_t ld_from, const int32_t * to, int64_t ld_to,
                                                     const int32_t * index, int64_t ld_index, const int32_t * count, int most) {
    constexpr int NB = D / 32, WORDS = D / 64;                           // 32-bit words of an eighth of a row
    const int s = blockIdx.z, i = blockIdx.x * 32 + (threadIdx.x >> 3), l = threadIdx.x & 7;
    if (i >= min(count[s], most)) return;                                // (the grid is rounded up: a count may say more than there is)
    const int32_t c = index[s * ld_index + i];
    if (c < 0 || c / KV4_CELLS >= ld_from || i / KV4_CELLS >= ld_to) return;
    const int64_t a = from[s * ld_from + c / KV4_CELLS], b = to[s * ld_to + i / KV4_CELLS];
    if (a < 0 || a >= n_pages || b < 0 || b >= n_pages) return;
    const int64_t page_bytes = (int64_t) chunks * kv4_chunk_bytes(D);
    const uint8_t * src = pages + a * page_bytes;
    uint8_t * dst = pages + b * page_bytes;
    const int ct = c % KV4_CELLS, it = i % KV4_CELLS;
    const int k_src = kv4_k_word(D, ct, 0, l * WORDS), k_dst = kv4_k_word(D, it, 0, l * WORDS);
    const int v_src = kv4_rows_bytes(D) + kv4_v_word(D, ct, l, 0), v_dst = kv4_rows_bytes(D) + kv4_v_word(D, it, l, 0);
    const int part = 2 * kv4_rows_bytes(D) + (l / NB) * kv4_scales_bytes(D), s_src = part + kv4_scale(D, ct, l % NB), s_dst = part + kv4_scale(D, it, l % NB);
    for (int r0 = blockIdx.y * KM_CHUNKS; r0 < chunks; r0 += gridDim.y * KM_CHUNKS) {
        uint32_t k[KM_CHUNKS][WORDS], v[KM_CHUNKS][WORDS];
        uint16_t sc[KM_CHUNKS];
#pragma unroll
        for (int r = 0; r < KM_CHUNKS; r++) {
            if (r0 + r >= chunks) continue;
            const uint8_t * p = src + (int64_t) (r0 + r) * kv4_chunk_bytes(D);
            if constexpr (WORDS == 2) {
                *reinterpret_cast<uint2 *>(k[r]) = *reinterpret_cast<const uint2 *>(p + k_src);
                *reinterpret_cast<uint2 *>(v[r]) = *reinterpret_cast<const uint2 *>(p + v_src);
            } else {
                k[r][0] = *reinterpret_cast<const uint32_t *>(p + k_src);
                v[r][0] = *reinterpret_cast<const uint32_t *>(p + v_src);
            }
            if (l < 2 * NB) sc[r] = *reinterpret_cast<const uint16_t *>(p + s_src);
        }
#pragma unroll
        for (int r = 0; r < KM_CHUNKS; r++) {
            if (r0 + r >= chunks) continue;
            uint8_t * p = dst + (int64_t) (r0 + r) * kv4_chunk_bytes(D);
            if constexpr (WORDS == 2) {
                *reinterpret_cast<uint2 *>(p + k_dst) = make_uint2(k[r][0], k[r][1]);
                *reinterpret_cast<uint2 *>(p + v_dst) = make_uint2(v[r][0], v[r][1]);
            } else {
                *reinterpret_cast<uint32_t *>(p + k_dst) = k[r][0];
                *reinterpret_cast<uint32_t *>(p + v_dst) = v[r][0];
            }
            if (l < 2 * NB) *reinterpret_cast<uint16_t *>(p + s_dst) = sc[r];
        }
    }
}

template <typename T>
int append(const Kv4 & cache, int D, const void * q, int64_t ldq, void * q_out, int64_t ldqo, const void * k, int64_t ldk, const void * v, int64_t ldv, int64_t n, int n_head,
           const int64_t * cells, const int32_t * pos, const float * q_norm, const float * k_norm, float eps, const Kv4Rope & rope, cudaStream_t st) {
    const AppendParams<T> p{cache, (const T *) q, (const T *) k, (const T *) v, (T *) q_out, ldq, ldqo, ldk, ldv, n_head, (int) n, cells, pos, q_norm, k_norm, eps};
    // Many tokens: two to a CTA, so that angles are made once, and four heads to a warp.  Few: a CTA has a token's heads in part, which makes the angles again for each.  us, many / few, bf16,
    // 32 heads over 8, with k_kv4_load: 150 tokens 10.8 / 8.7, 200 10.9 / 10.7, 300 12.2 / 12.9, 600 15 / 20
    if (n >= KA_MANY * sm_count()) {
        const unsigned grid = (unsigned) ((n + 1) / 2);
        if (D == 128) k_kv4_append<T, 128, 2, 4><<<grid, KA_THREADS, 0, st>>>(p, rope);
        else k_kv4_append<T, 64, 2, 4><<<grid, KA_THREADS, 0, st>>>(p, rope);
    } else {
        const int64_t items = (n_head + 2 * (int64_t) cache.n_head_kv + 32 / (D / 4) - 1) / (32 / (D / 4)), parts = (items + KA_WARPS - 1) / KA_WARPS, most = (4 * sm_count() + n - 1) / n;
        const dim3 grid((unsigned) n, (unsigned) (parts < most ? parts : most));
        if (D == 128) k_kv4_append<T, 128, 1, 1><<<grid, KA_THREADS, 0, st>>>(p, rope);
        else k_kv4_append<T, 64, 1, 1><<<grid, KA_THREADS, 0, st>>>(p, rope);
    }
    return (int) cudaGetLastError();
}
template <typename T>
int load(const Kv4 & cache, int D, const int64_t * cells, int64_t n, void * k, int64_t ldk, void * v, int64_t ldv, cudaStream_t st) {
    const int64_t threads = n * cache.n_head_kv * (D / 4);
    const unsigned grid = (unsigned) ((threads + 255) / 256);
    if (D == 128) k_kv4_load<T, 128><<<grid, 256, 0, st>>>(cache, cells, n, (T *) k, ldk, (T *) v, ldv);
    else k_kv4_load<T, 64><<<grid, 256, 0, st>>>(cache, cells, n, (T *) k, ldk, (T *) v, ldv);
    return (int) cudaGetLastError();
}

}  // namespace

int launch_kv4_append(const Kv4 & cache, int D, int type, const void * q, int64_t ldq, void * q_out, int64_t ldqo, const void * k, int64_t ldk, const void * v, int64_t ldv, int64_t n,
                      int n_head, const int64_t * cells, const int32_t * pos, const float * q_norm, const float * k_norm, float eps, const Kv4Rope & rope, cudaStream_t st) {
    const auto f = type == PB200_TYPE_F32 ? append<float> : type == PB200_TYPE_F16 ? append<__half> : append<__nv_bfloat16>;
    return f(cache, D, q, ldq, q_out, ldqo, k, ldk, v, ldv, n, n_head, cells, pos, q_norm, k_norm, eps, rope, st);
}

int launch_kv4_load(const Kv4 & cache, int D, int type, const int64_t * cells, int64_t n, void * k, int64_t ldk, void * v, int64_t ldv, cudaStream_t st) {
    const auto f = type == PB200_TYPE_F32 ? load<float> : type == PB200_TYPE_F16 ? load<__half> : load<__nv_bfloat16>;
    return f(cache, D, cells, n, k, ldk, v, ldv, st);
}

int launch_kv4_copy_pages(uint8_t * pages, int64_t page_bytes, const int32_t * src, const int32_t * dst, int n, cudaStream_t st) {
    for (int at = 0; at < n; at += KC_PAIRS) {
        CopyPairs p{};
        const int m = n - at < KC_PAIRS ? n - at : KC_PAIRS;
        for (int i = 0; i < m; i++) { p.src[i] = src[at + i]; p.dst[i] = dst[at + i]; }
        const int64_t want = (page_bytes / 16 + KC_ONCE * 256 - 1) / (KC_ONCE * 256), most = (16 * sm_count() + m - 1) / m;
        k_kv4_copy_pages<<<dim3((unsigned) (want < most ? want : most), (unsigned) m), 256, 0, st>>>(pages, page_bytes, p);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return (int) e;
    }
    return 0;
}

int launch_kv4_compact(uint8_t * pages, int64_t n_pages, int rows, int D, int n_seq, const int32_t * from, int64_t ld_from, const int32_t * to, int64_t ld_to, const int32_t * index,
                       int64_t ld_index, const int32_t * count, int most, cudaStream_t st) {
    const dim3 grid((unsigned) (((int64_t) most + 31) / 32), (unsigned) ((rows + KM_CHUNKS - 1) / KM_CHUNKS), (unsigned) n_seq);
    if (D == 128) k_kv4_compact<128><<<grid, 256, 0, st>>>(pages, n_pages, rows, from, ld_from, to, ld_to, index, ld_index, count, most);
    else k_kv4_compact<64><<<grid, 256, 0, st>>>(pages, n_pages, rows, from, ld_from, to, ld_to, index, ld_index, count, most);
    return (int) cudaGetLastError();
}

}  // namespace pb
