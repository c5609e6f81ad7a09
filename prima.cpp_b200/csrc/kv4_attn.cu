// prima.cpp_b200/csrc/kv4_attn.cu — attention over the 4-bit cache (kv4.cuh).
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/prima_b200.h"
#include "kv4_attn.cuh"

namespace pb {
namespace {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float * p, float x) { *p = x; }
__device__ __forceinline__ void put(__half * p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void put(__nv_bfloat16 * p, float x) { *p = __float2bfloat16_rn(x); }

// A warp to a (token, head): scores of 32 cells at a time, one to a lane; running maximum and sum; a lane keeps D / 32 numbers of the output.
template <typename T, int D>
__global__ void __launch_bounds__(128) k_kv4_attn_warp(const __grid_constant__ Kv4Attn A) {
    __shared__ float q_s[4][D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t item = (int64_t) blockIdx.x * 4 + warp;
    if (item >= A.n_tokens * A.n_head) return;
    const int64_t tok = item / A.n_head;
    const int head = (int) (item % A.n_head), hk = head / A.group;
    int lo = 0, hi = A.n_seq;          // the sequence: last s with q_start[s] <= tok
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (A.q_start[mid] <= tok) lo = mid; else hi = mid;
    }
    const int s = lo;
    if (tok < A.q_start[s] || tok >= A.q_start[s + 1] || tok - A.q_start[s] >= A.max_q) return;
    const int p = A.kv_len[s] - A.q_start[s + 1] + (int) tok;
    for (int d = lane; d < D; d += 32) q_s[warp][d] = to_f32(((const T *) A.q)[tok * A.ldq + (int64_t) head * D + d]) * A.scale;
    __syncwarp();
    float m = -INFINITY, l = 0.f, o[D / 32];
    for (int i = 0; i < D / 32; i++) o[i] = 0.f;
    for (int64_t c0 = 0; c0 <= p; c0 += 32) {
        if (A.window > 0 && c0 >= A.first && p - (c0 + 31) >= A.window) continue;
        const int64_t pi = c0 / KV4_CELLS;
        const int64_t page = pi < A.table_ld ? A.table[s * A.table_ld + pi] : -1;
        if (page < 0 || page >= A.cache.n_pages) continue;
        const uint8_t * chunk = kv4_chunk<D>(A.cache, page, hk);
        const int t = (int) (c0 % KV4_CELLS) + lane;
        const int64_t cell = c0 + lane;
        const bool see = cell <= p && (A.window <= 0 || p - cell < A.window || cell < A.first);
        float sc = -INFINITY;
        if (see) {
            sc = 0.f;
            for (int b = 0; b < D / 32; b++) {
                float part = 0.f;
                for (int c = 0; c < 4; c++) {
                    const uint32_t w = *(const uint32_t *) (chunk + kv4_k_word(D, t, c, b));
                    for (int e = 0; e < 8; e++) part += q_s[warp][32 * b + 8 * c + e] * (float) ((int) (w >> (4 * (e / 2) + 16 * (e % 2)) & 15) - 8);
                }
                sc += part * __half2float(*(const __half *) (chunk + 2 * kv4_rows_bytes(D) + kv4_scale(D, t, b)));
            }
        }
        const float mn = fmaxf(m, warp_max(sc));
        if (!__any_sync(0xffffffffu, see)) continue;
        const float f = expf(m - mn), e = see ? expf(sc - mn) : 0.f;
        l = l * f + warp_sum(e);
        m = mn;
        for (int i = 0; i < D / 32; i++) o[i] *= f;
        for (int j = 0; j < 32; j++) {
            const float w = __shfl_sync(0xffffffffu, e, j);
            if (w == 0.f) continue;
            const int tj = t - lane + j;
            for (int i = 0; i < D / 32; i++) {
                const uint32_t h = *(const uint16_t *) (chunk + kv4_rows_bytes(D) + kv4_v_word(D, tj, lane / 4, i));
                const float sv = __half2float(*(const __half *) (chunk + 2 * kv4_rows_bytes(D) + kv4_scales_bytes(D) + kv4_scale(D, tj, i)));
                o[i] += w * ((float) ((int) (h >> (4 * (lane & 3)) & 15) - 8) * sv);
            }
        }
    }
    for (int i = 0; i < D / 32; i++) put((T *) A.out + tok * A.ldo + (int64_t) head * D + 32 * i + lane, l == 0.f ? 0.f : o[i] / l);
}

template <typename T>
int attn(const Kv4Attn & a, int D, cudaStream_t st) {
    const int64_t items = a.n_tokens * a.n_head;
    const unsigned grid = (unsigned) ((items + 3) / 4);
    if (D == 128) k_kv4_attn_warp<T, 128><<<grid, 128, 0, st>>>(a);
    else k_kv4_attn_warp<T, 64><<<grid, 128, 0, st>>>(a);
    return (int) cudaGetLastError();
}

}  // namespace

size_t kv4_attn_workspace(int D, int, int) { return KV4_COUNTERS * sizeof(int) + kv4_rows_workspace(D); }

int launch_kv4_attn(const Kv4Attn & a, int D, int type, void * ws, cudaStream_t st) {
    return launch_kv4_attn_rows(a, D, type, 1 << 30, (int *) ws, (char *) ws + KV4_COUNTERS * sizeof(int), st);
}

}  // namespace pb
