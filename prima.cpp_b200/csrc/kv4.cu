// prima.cpp_b200/csrc/kv4.cu — what writes and moves the cells of the 4-bit cache (kv4.cuh): rows of a step into their cells with the norms of queries and
// keys and the rotation on the way, their values back, pages of a fork, cells that are kept.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/prima_b200.h"
#include "kv4.cuh"

namespace pb {
namespace {

constexpr int KA_THREADS = 256;

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

// A CTA takes a token and a part of its rows (heads of q, k, v), a quarter of a head's numbers at a time to a thread: D / 4 lanes hold a row, four neighbouring
// numbers each.  What decides which of 16 steps a number falls to is computed so that it does not depend on an order: the mean of squares and the angles in
// 64 bits, rounded once, products and sums of the rotation in 32 bits without contraction.
template <typename T, int D>
__global__ void __launch_bounds__(KA_THREADS) k_kv4_append(const __grid_constant__ AppendParams<T> P, const __grid_constant__ Kv4Rope R) {
    constexpr int LPR = D / 4, NB = D / 32;       // lanes to a row
    __shared__ float2 cs[D / 2];
    const int t = blockIdx.x, lane = threadIdx.x & 31;
    const int pairs = R.n_dims / 2;
    if (threadIdx.x < pairs) {
        const double a = (double) P.pos[t] * R.w[threadIdx.x] / (R.freq_factors ? (double) R.freq_factors[threadIdx.x] : 1.0);
        double s, c;
        sincos(a, &s, &c);
        cs[threadIdx.x] = make_float2(__fmul_rn((float) c, R.mscale), __fmul_rn((float) s, R.mscale));
    }
    __syncthreads();
    const int64_t cell = P.cells[t];
    const bool stored = cell >= 0 && cell < P.cache.n_pages * KV4_CELLS;
    const int hk = P.cache.n_head_kv, rows = P.n_head + 2 * hk;
    const int sub = lane / LPR, l = lane % LPR, d = 4 * l;
    const int per = 32 / LPR * (KA_THREADS / 32);
    for (int r0 = blockIdx.y * per; r0 < rows; r0 += gridDim.y * per) {
        const int row = r0 + (threadIdx.x >> 5) * (32 / LPR) + sub;
        const bool mine = row < rows;
        const int kind = !mine ? 3 : row < P.n_head ? 0 : row < P.n_head + hk ? 1 : 2;
        const int head = kind == 0 ? row : kind == 1 ? row - P.n_head : row - P.n_head - hk;
        const T * src = kind == 0 ? P.q + t * P.ldq : kind == 1 ? P.k + t * P.ldk : P.v + t * P.ldv;
        float4 x4 = make_float4(0.f, 0.f, 0.f, 0.f);
        if (mine) x4 = load4(src + (int64_t) head * D + d);
        float x[4] = {x4.x, x4.y, x4.z, x4.w};
        const float * w = kind == 0 ? P.q_norm : kind == 1 ? P.k_norm : nullptr;
        if (P.q_norm || P.k_norm) {
            double sum = 0.0;
#pragma unroll
            for (int i = 0; i < 4; i++) sum += (double) x[i] * (double) x[i];
#pragma unroll
            for (int o = LPR / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (w) {
                const float r = (float) (1.0 / sqrt(sum / D + (double) P.eps));
                const float4 w4 = load4(w + d);
                x[0] = __fmul_rn(__fmul_rn(x[0], r), w4.x);
                x[1] = __fmul_rn(__fmul_rn(x[1], r), w4.y);
                x[2] = __fmul_rn(__fmul_rn(x[2], r), w4.z);
                x[3] = __fmul_rn(__fmul_rn(x[3], r), w4.w);
            }
        }
        if (pairs > 0) {
            const int half = pairs / 4;            // lanes between the two of a pair (mode 2)
            float y[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float o = __shfl_sync(0xffffffffu, x[i], R.mode == 0 ? lane ^ 0 : d < pairs ? lane + half : lane - half);
                y[i] = R.mode == 0 ? x[i ^ 1] : o;
            }
            if (kind < 2 && d < 2 * pairs) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const bool first = R.mode == 0 ? (i & 1) == 0 : d < pairs;
                    const float2 a = cs[R.mode == 0 ? (d + i) / 2 : first ? d + i : d + i - pairs];
                    x[i] = first ? __fsub_rn(__fmul_rn(x[i], a.x), __fmul_rn(y[i], a.y)) : __fadd_rn(__fmul_rn(y[i], a.y), __fmul_rn(x[i], a.x));
                }
            }
        }
        if (kind == 0) store4(P.q_out + t * P.ldqo + (int64_t) head * D + d, make_float4(x[0], x[1], x[2], x[3]));
        // keys and values: the block's number of largest magnitude (of several, the first), scale, bits
        float most = 0.f;
        bool any = false;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[i] = kv4_finite(x[i]);
            if (fabsf(x[i]) > fabsf(most) || i == 0) most = x[i];
        }
        float top = fabsf(most);
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        any = fabsf(most) == top;
        const uint32_t who = __ballot_sync(0xffffffffu, any) & (0xffu << (lane & 24));
        const float scale = kv4_scale_of(__shfl_sync(0xffffffffu, most, __ffs((int) who) - 1));
        uint32_t n[4];
#pragma unroll
        for (int i = 0; i < 4; i++) n[i] = kv4_bits_of(x[i], scale);
        const int b = d / 32;
        uint32_t word = (n[0] | n[1] << 16 | n[2] << 4 | n[3] << 20) << (8 * (l & 1));
        word |= __shfl_xor_sync(0xffffffffu, word, 1);
        if ((kind == 1 || kind == 2) && stored) {
            const int at = (int) (cell % KV4_CELLS);
            uint8_t * chunk = kv4_chunk<D>(P.cache, cell / KV4_CELLS, head);
            if (kind == 1) {
                if ((l & 1) == 0) *reinterpret_cast<uint32_t *>(chunk + kv4_k_word(D, at, (d / 8) % 4, b)) = word;
            } else {
                *reinterpret_cast<uint16_t *>(chunk + kv4_rows_bytes(D) + kv4_v_word(D, at, (d / 4) % 8, b)) = (uint16_t) (n[0] | n[1] << 4 | n[2] << 8 | n[3] << 12);
            }
            if ((l & 7) == 0)
                *reinterpret_cast<__half *>(chunk + 2 * kv4_rows_bytes(D) + (kind == 2 ? kv4_scales_bytes(D) : 0) + kv4_scale(D, at, b)) = __float2half_rn(scale);
        }
        (void) NB;
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

constexpr int KC_PAIRS = 256;
struct CopyPairs { int32_t src[KC_PAIRS], dst[KC_PAIRS]; };
__global__ void __launch_bounds__(256) k_kv4_copy_pages(uint8_t * pages, int64_t page_bytes, const __grid_constant__ CopyPairs p) {
    const uint4 * s = reinterpret_cast<const uint4 *>(pages + p.src[blockIdx.y] * page_bytes);
    uint4 * d = reinterpret_cast<uint4 *>(pages + p.dst[blockIdx.y] * page_bytes);
    const int64_t n = page_bytes / 16;
    for (int64_t i = (int64_t) blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t) gridDim.x * 256) d[i] = s[i];
}

template <int D>
__global__ void __launch_bounds__(256) k_kv4_compact(uint8_t * pages, int64_t n_pages, int rows, const int32_t * from, int64_t ld_from, const int32_t * to, int64_t ld_to,
                                                     const int32_t * index, int64_t ld_index, const int32_t * count) {
    constexpr int NB = D / 32;
    const int s = blockIdx.z, row = blockIdx.y;
    const int i = blockIdx.x * 16 + (threadIdx.x >> 4), l = threadIdx.x & 15;     // 16 threads to a cell
    if (i >= count[s]) return;
    const int32_t c = index[s * ld_index + i];
    if (c < 0 || c / KV4_CELLS >= ld_from || i / KV4_CELLS >= ld_to) return;
    const int64_t a = from[s * ld_from + c / KV4_CELLS], b = to[s * ld_to + i / KV4_CELLS];
    if (a < 0 || a >= n_pages || b < 0 || b >= n_pages) return;
    const int64_t page_bytes = (int64_t) rows * kv4_chunk_bytes(D);
    const uint8_t * src = pages + a * page_bytes + (int64_t) row * kv4_chunk_bytes(D);
    uint8_t * dst = pages + b * page_bytes + (int64_t) row * kv4_chunk_bytes(D);
    const int ct = c % KV4_CELLS, it = i % KV4_CELLS;
    for (int w = l; w < D / 8; w += 16) {
        *reinterpret_cast<uint32_t *>(dst + kv4_k_word(D, it, 0, w)) = *reinterpret_cast<const uint32_t *>(src + kv4_k_word(D, ct, 0, w));
        for (int h = 2 * w; h < 2 * w + 2; h++)
            *reinterpret_cast<uint16_t *>(dst + kv4_rows_bytes(D) + kv4_v_word(D, it, h / NB, h % NB)) =
                *reinterpret_cast<const uint16_t *>(src + kv4_rows_bytes(D) + kv4_v_word(D, ct, h / NB, h % NB));
    }
    if (l < 2 * NB) {
        const int part = 2 * kv4_rows_bytes(D) + (l / NB) * kv4_scales_bytes(D);
        *reinterpret_cast<uint16_t *>(dst + part + kv4_scale(D, it, l % NB)) = *reinterpret_cast<const uint16_t *>(src + part + kv4_scale(D, ct, l % NB));
    }
}

template <typename T>
int append(const Kv4 & cache, int D, const void * q, int64_t ldq, void * q_out, int64_t ldqo, const void * k, int64_t ldk, const void * v, int64_t ldv, int64_t n, int n_head,
           const int64_t * cells, const int32_t * pos, const float * q_norm, const float * k_norm, float eps, const Kv4Rope & rope, cudaStream_t st) {
    const AppendParams<T> p{cache, (const T *) q, (const T *) k, (const T *) v, (T *) q_out, ldq, ldqo, ldk, ldv, n_head, (int) n, cells, pos, q_norm, k_norm, eps};
    const int per = 32 / (D / 4) * (KA_THREADS / 32), rows = n_head + 2 * cache.n_head_kv;
    const dim3 grid((unsigned) n, (unsigned) ((rows + per - 1) / per < 1024 ? (rows + per - 1) / per : 1024));
    if (D == 128) k_kv4_append<T, 128><<<grid, KA_THREADS, 0, st>>>(p, rope);
    else k_kv4_append<T, 64><<<grid, KA_THREADS, 0, st>>>(p, rope);
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
        const int64_t want = (page_bytes / 16 + 255) / 256;
        k_kv4_copy_pages<<<dim3((unsigned) (want < 64 ? want : 64), (unsigned) m), 256, 0, st>>>(pages, page_bytes, p);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return (int) e;
    }
    return 0;
}

int launch_kv4_compact(uint8_t * pages, int64_t n_pages, int rows, int D, int n_seq, const int32_t * from, int64_t ld_from, const int32_t * to, int64_t ld_to, const int32_t * index,
                       int64_t ld_index, const int32_t * count, int most, cudaStream_t st) {
    const dim3 grid((unsigned) ((most + 15) / 16), (unsigned) rows, (unsigned) n_seq);
    if (D == 128) k_kv4_compact<128><<<grid, 256, 0, st>>>(pages, n_pages, rows, from, ld_from, to, ld_to, index, ld_index, count);
    else k_kv4_compact<64><<<grid, 256, 0, st>>>(pages, n_pages, rows, from, ld_from, to, ld_to, index, ld_index, count);
    return (int) cudaGetLastError();
}

}  // namespace pb
