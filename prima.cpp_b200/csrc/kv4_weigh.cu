// prima.cpp_b200/csrc/kv4_weigh.cu — what the cells of the 4-bit cache (kv4.cuh) are worth: their attention weights, added up over queries and heads.
//
// Mathematics.  sums[j] = decay * old[j] + sum over queries t and heads h that see cell j of 2^(c q_th . k_j - L_th): L is the logarithm of the row's sum, which attention left, so that no row
// has to be looked at as a whole: a cell's sum is that of its own column.  Scores are m16n8k16 products, cells x rows: a thread holds two rows' scores of a cell next to each other, and adds
// them up without asking others.  Keys are f16 numbers exactly and go to registers once for all rows; a query row is f16 times a power of two (F32: two of them, 22 bits, low parts first).
//
// Work.  An item is 256 cells of a sequence, 32 to each of a CTA's warps.  A cluster has an item; its CTAs share the kv heads, and the rows in blocks of 64; their sums meet in shared memory, in
// the CTAs' order (equal calls give equal bits).
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cfloat>
#include <type_traits>

#include "../../include/prima_b200.h"
#include "cluster.cuh"
#include "kv4_attn.cuh"

namespace pb {
namespace {

constexpr int KW_WARPS = 8, KW_THREADS = 32 * KW_WARPS, KW_CELLS = 32 * KW_WARPS, KW_ROWS = 64;

// rows of a block: f16 numbers (F32: high, then low parts), in rows that lie 64 bytes further on than they are long: the eight rows of a product are in different banks
template <int D, bool F32> struct __align__(16) KwSmem {
    __align__(16) uint8_t q[F32 ? 2 : 1][KW_ROWS][2 * D + 64];
    float2 row[KW_ROWS];       // of a score to the power of two, and the logarithm of the row's sum
    int pos[KW_ROWS];
    float part[2][KW_CELLS];   // what the cluster's CTAs add up
    int ends[KW_THREADS], warp[KW_WARPS];
};

__device__ __forceinline__ uint32_t hu(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
__device__ __forceinline__ __half2 uh(uint32_t u) { return *reinterpret_cast<__half2 *>(&u); }
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T, int D>
__global__ void __launch_bounds__(KW_THREADS, 2) k_kv4_weigh(const __grid_constant__ Kv4Weigh W) {
    constexpr bool F32 = std::is_same<T, float>::value;
    constexpr int NB = D / 32, LO = F32 ? 2 : 1;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    KwSmem<D, F32> & S = *reinterpret_cast<KwSmem<D, F32> *>(smem_raw);
    const Kv4Attn & A = W.attn;
    const int tid = threadIdx.x, lane = tid & 31, warp = uniform_warp(), g = lane >> 2, c = lane & 3, hks = A.cache.n_head_kv;
    const int ctas = (int) cluster_size(), rank = (int) cluster_rank();

    auto length = [&](int s) { return s < A.n_seq ? (int) max((int64_t) 0, min((int64_t) A.kv_len[s], W.ld_sums)) : 0; };
    // items of 256 sequences at a time: where each one's end; the items in front of them
    int at = -1, before = 0, all = 0;
    auto scan = [&](int s0) {
        int x = (length(s0 + tid) + KW_CELLS - 1) / KW_CELLS;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        __syncthreads();
        if (lane == 31) S.warp[warp] = x;
        __syncthreads();
        all = 0;
#pragma unroll
        for (int w = 0; w < KW_WARPS; w++) {
            if (w < warp) x += S.warp[w];
            all += S.warp[w];
        }
        S.ends[tid] = x;
        at = s0;
        __syncthreads();
    };
    int flip = 0;
    for (int item = blockIdx.x / ctas;; item += gridDim.x / ctas) {
        // ---- which cells of which sequence (ascending: those of sequences further on) ----
        if (at < 0) scan(0);
        while (item - before >= all) {
            before += all;
            if (at + KW_THREADS >= A.n_seq) {
                cluster_sync();                             // nobody reads a CTA's sums that has ended
                return;
            }
            scan(at + KW_THREADS);
        }
        const int k = __syncthreads_count(S.ends[tid] <= item - before), s = at + k;
        const int base = (item - before - (k > 0 ? S.ends[k - 1] : 0)) * KW_CELLS, len = length(s);

        // ---- the rows that see any of them ----
        const int64_t q0 = A.q_start[s], q1 = A.q_start[s + 1];
        const bool some = q0 >= 0 && q1 > q0 && q1 <= A.n_tokens;
        const int n_all = some ? (int) (q1 - q0) : 0, n_q = min(n_all, A.max_q), p0 = max(A.kv_len[s], 0) - n_all;
        int t_lo = min(n_q, max(0, base - p0)), t_hi = n_q;
        if (A.window > 0 && base >= A.first) t_hi = (int) max((int64_t) t_lo, min((int64_t) n_q, (int64_t) base + KW_CELLS - 1 + A.window - p0));
        const int r_lo = t_lo * A.group, rows = t_hi * A.group - r_lo, blocks = (rows + KW_ROWS - 1) / KW_ROWS, units = hks * blocks;
        const int u0 = (int) ((int64_t) units * rank / ctas), u1 = (int) ((int64_t) units * (rank + 1) / ctas);

        // ---- this warp's cells: page, keys of a kv head ----
        const int cell0 = base + 32 * warp, in_page = cell0 % KV4_CELLS;
        const int page_at = cell0 / KV4_CELLS;
        int page = -1;
        if (cell0 < len && page_at < A.table_ld) {
            page = A.table[s * A.table_ld + page_at];
            if (page >= A.cache.n_pages) page = -1;
        }
        uint32_t kf[2][NB][2][4];                           // eights of cells 16 m + g (+ 8): block, half of the eight numbers
        float sum[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
        int held = -1;
        for (int u = u0; u < u1; u++) {
            const int hk = u / blocks, row0 = r_lo + (u - hk * blocks) * KW_ROWS, n = min(KW_ROWS, r_lo + rows - row0);
            if (held != hk && page >= 0) {
                const uint8_t * chunk = kv4_chunk<D>(A.cache, page, hk), * scales = chunk + 2 * kv4_rows_bytes(D);
#pragma unroll
                for (int m = 0; m < 2; m++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int t = in_page + 16 * m + 8 * h + g;
                        uint32_t w[NB], d[NB];
                        if constexpr (NB == 4) {
                            *reinterpret_cast<uint4 *>(w) = *reinterpret_cast<const uint4 *>(chunk + t * (D / 2) + 16 * c);
                            *reinterpret_cast<uint4 *>(d) = *reinterpret_cast<const uint4 *>(scales + kv4_scale(D, t & ~1, 0));
                        } else {
                            *reinterpret_cast<uint2 *>(w) = *reinterpret_cast<const uint2 *>(chunk + t * (D / 2) + 8 * c);
                            *reinterpret_cast<uint2 *>(d) = *reinterpret_cast<const uint2 *>(scales + kv4_scale(D, t & ~1, 0));
                        }
#pragma unroll
                        for (int b = 0; b < NB; b++) {
                            const __half2 sc = uh(__byte_perm(d[b], 0u, t & 1 ? 0x3232u : 0x1010u)), e = __float2half2_rn(1032.f), o = __float2half2_rn(72.f);
                            const uint32_t x = w[b], y = w[b] >> 8;
                            kf[m][b][0][h] = hu(__hmul2(__hsub2(uh((x & 0x000f000fu) | 0x64006400u), e), sc));
                            kf[m][b][0][2 + h] = hu(__hmul2(__hsub2(uh((x & 0x00f000f0u) | 0x54005400u), o), sc));
                            kf[m][b][1][h] = hu(__hmul2(__hsub2(uh((y & 0x000f000fu) | 0x64006400u), e), sc));
                            kf[m][b][1][2 + h] = hu(__hmul2(__hsub2(uh((y & 0x00f000f0u) | 0x54005400u), o), sc));
                        }
                    }
                held = hk;
            }
            // the block's rows: four threads to a row, 32 numbers of one block each at a time
            __syncthreads();
            {
                const int r = tid >> 2, quarter = tid & 3, row = row0 + r, t = row / A.group, head = hk * A.group + row - t * A.group;
                const bool have = r < n;
                constexpr int EACH = D / 4;
                float x[EACH], top = 0.f;
                const T * src = (const T *) A.q + (q0 + t) * A.ldq + (int64_t) head * D + quarter * EACH;
#pragma unroll
                for (int i = 0; i < EACH; i += 4) {
                    const float4 v = have ? load4(src + i) : make_float4(0.f, 0.f, 0.f, 0.f);
                    x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
                }
                const float lse = have ? W.lse[(q0 + t) * W.ld_lse + head] : -INFINITY;
#pragma unroll
                for (int i = 0; i < EACH; i++) top = fmaxf(top, fabsf(x[i]));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                // the row's power of two: its largest number comes to 2^13 .. 2^14
                const int ex = top > 0.f && top < INFINITY ? min(126, 140 - (int) (__float_as_uint(top) >> 23)) : 0;
                const float up = __int_as_float((ex + 127) << 23) * (A.scale < 0.f ? -1.f : 1.f);
#pragma unroll
                for (int i = 0; i < EACH; i += 8) {
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float a = x[i + 2 * e] * up, b = x[i + 2 * e + 1] * up;
                        const __half2 h = __floats2half2_rn(a, b);
                        hi[e] = hu(h);
                        if constexpr (F32) {
                            const float2 back = __half22float2(h);
                            lo[e] = hu(__floats2half2_rn(a - back.x, b - back.y));
                        }
                    }
                    *reinterpret_cast<uint4 *>(&S.q[0][r][2 * (quarter * EACH + i)]) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    if constexpr (F32) *reinterpret_cast<uint4 *>(&S.q[LO - 1][r][2 * (quarter * EACH + i)]) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
                if (quarter == 0) {
                    // a row that saw nothing has no weights
                    S.row[r] = make_float2(fmaxf(fabsf(A.scale) * 1.4426950408889634f * __int_as_float((127 - ex) << 23), FLT_MIN), lse == -INFINITY ? INFINITY : lse * 1.4426950408889634f);
                    S.pos[r] = have ? p0 + t : -1;
                }
            }
            __syncthreads();
            const int p_lo = p0 + row0 / A.group, p_hi = p0 + (row0 + n - 1) / A.group;
            if (page < 0 || cell0 > p_hi) continue;
            const bool whole = cell0 + 31 <= p_lo && (A.window <= 0 || p_hi - cell0 < A.window || cell0 + 31 < A.first);
#pragma unroll 1
            for (int j = 0; j < n; j += 8) {
                float acc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
                for (int part = LO - 1; part >= 0; part--)
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        const uint4 q = *reinterpret_cast<const uint4 *>(&S.q[part][j + g][64 * b + 16 * c]);
#pragma unroll
                        for (int m = 0; m < 2; m++) {
                            mma16816(acc[m], kf[m][b][0], q.x, q.y);
                            mma16816(acc[m], kf[m][b][1], q.z, q.w);
                        }
                    }
                const float4 r = *reinterpret_cast<const float4 *>(&S.row[j + 2 * c]);
                float e[2][4];
#pragma unroll
                for (int m = 0; m < 2; m++)
#pragma unroll
                    for (int i = 0; i < 4; i++) e[m][i] = ex2(fmaf(acc[m][i], i & 1 ? r.z : r.x, i & 1 ? -r.w : -r.y));
                if (!whole) {
                    const int2 pos = *reinterpret_cast<const int2 *>(&S.pos[j + 2 * c]);
#pragma unroll
                    for (int m = 0; m < 2; m++)
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int cell = cell0 + 16 * m + 8 * (i >> 1) + g, p = i & 1 ? pos.y : pos.x;
                            if (!(cell <= p && (A.window <= 0 || p - cell < A.window || cell < A.first))) e[m][i] = 0.f;
                        }
                }
#pragma unroll
                for (int m = 0; m < 2; m++) {
                    sum[m][0] += e[m][0] + e[m][1];
                    sum[m][1] += e[m][2] + e[m][3];
                }
            }
        }
        // ---- the cluster's sums ----
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                float x = sum[m][h];
                x += __shfl_xor_sync(0xffffffffu, x, 1);
                x += __shfl_xor_sync(0xffffffffu, x, 2);
                if (c == 0) S.part[flip][32 * warp + 16 * m + 8 * h + g] = x;
            }
        cluster_sync();                                     // (of the item behind the next one's, nobody reads these any more)
        for (int i = rank * KW_CELLS / ctas + tid; i < (rank + 1) * KW_CELLS / ctas; i += KW_THREADS) {
            float x = 0.f;
            for (int r = 0; r < ctas; r++) x += remote(&S.part[flip][i], r);
            const int64_t j = base + i;
            if (j < len) W.sums[s * W.ld_sums + j] = W.old ? fmaf(W.decay, W.old[s * W.ld_old + j], x) : x;
        }
        flip ^= 1;
    }
}

template <typename T, int D>
int weigh_launch(const Kv4Weigh & w, cudaStream_t st) {
    constexpr size_t smem = sizeof(KwSmem<D, std::is_same<T, float>::value>);
    static FuncAttrCache cache;
    cudaError_t e = ensure_dyn_smem(cache, (const void *) k_kv4_weigh<T, D>, smem, false);
    if (e != cudaSuccess) return (int) e;
    const int64_t rows = std::min<int64_t>(w.attn.max_q, w.attn.n_tokens) * w.attn.group, units = w.attn.cache.n_head_kv * ((rows + KW_ROWS - 1) / KW_ROWS);
    const int ctas = units >= 8 ? 8 : units >= 4 ? 4 : units >= 2 ? 2 : 1;
    return (int) launch_clusters(k_kv4_weigh<T, D>, std::max(1, 2 * sm_count() / ctas), ctas, KW_THREADS, smem, false, st, w);
}

}  // namespace

int launch_kv4_weigh(const Kv4Weigh & w, int D, int type, cudaStream_t st) {
    if (D == 128) return type == PB200_TYPE_F32 ? weigh_launch<float, 128>(w, st) : type == PB200_TYPE_F16 ? weigh_launch<__half, 128>(w, st) : weigh_launch<__nv_bfloat16, 128>(w, st);
    return type == PB200_TYPE_F32 ? weigh_launch<float, 64>(w, st) : type == PB200_TYPE_F16 ? weigh_launch<__half, 64>(w, st) : weigh_launch<__nv_bfloat16, 64>(w, st);
}

}  // namespace pb
