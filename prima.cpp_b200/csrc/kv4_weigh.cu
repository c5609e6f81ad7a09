// prima.cpp_b200/csrc/kv4_weigh.cu — what the cells of the 4-bit cache (kv4.cuh) are worth: their attention weights, added up over queries and heads.
//
// Mathematics.  sums[j] = decay * old[j] + sum over queries t and heads h that see cell j of 2^(c q_th . k_j - L_th): L is the logarithm of the row's sum, which attention left, so that no row
// has to be looked at as a whole: a cell's sum is that of its own column.  Scores are m16n8k16 products, cells x rows: a thread holds two rows' scores of a cell next to each other, and adds
// them up without asking others.  Keys are f16 numbers exactly and go to registers once for all rows; a query row is f16 times a power of two (F32: two of them, 22 bits, low parts first; many rows of F16 are as they are).
//
// Work.  Two kernels.  Few rows (tokens that decode): keys stream through shared memory, rows stay there.  Many rows: an item is 256, 128 or 64 cells of a sequence, 32 to each of a CTA's warps (128 and
// 64: two or four warps have the same cells, and each a part of the rows).  A cluster has an item; its CTAs share the kv heads, and the rows in blocks of 64; their sums meet in shared memory, in the
// CTAs' order (equal calls give equal bits).
//
// Bound: latency, no pipe is full.  Few rows: a key's numbers are taken apart once for up to 16 rows, by the 16 warps that an SM has room for (32 sequences of up to 8192 cells 33 us; their keys' bytes take 12: issue
// slots 40 %, DRAM 28 %).  Many rows (tensor pipe 19 %, XU 29 %, issue slots 26 %): of a block of 64 rows 1.2 us go into
// loading and converting, 2 into the products' chains and exponentials (64 queries of 32 heads behind 16 000 cells 41 us, 0.12 of the tensor cores' rate; 2048 of a prompt, on 128 CTAs, 259).
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
struct KwSplit { int cells, cuts; };     // of an item: 32 to a warp; so many warps have the same cells, each its part of a block's rows

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
// ORDERED: not moved among others; left to itself the compiler mixes products whose parts do not all fit into registers
template <bool ORDERED = false>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
#define PB_MMA "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
    if constexpr (ORDERED) asm volatile(PB_MMA : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else asm(PB_MMA : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
#undef PB_MMA
}

// ---- a query row in shared memory, a part of it to each of four threads next to each other ----
// its power of two: the largest number comes to 2^13 .. 2^14
template <int EACH>
__device__ __forceinline__ float row_power(const float (&x)[EACH]) {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < EACH; i++) top = fmaxf(top, fabsf(x[i]));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int ex = top > 0.f && top < INFINITY ? min(126, 140 - (int) (__float_as_uint(top) >> 23)) : 0;
    return __int_as_float((ex + 127) << 23);
}
template <typename T, int EACH, bool RAW = false>      // RAW: pairs 1 and 3 of eight numbers a 16th
__device__ __forceinline__ void row_store(const float (&x)[EACH], float up, uint8_t * high, uint8_t * low) {
#pragma unroll
    for (int i = 0; i < EACH; i += 8) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float a = x[i + 2 * e] * up, b = x[i + 2 * e + 1] * up;
            const __half2 h = __floats2half2_rn(a, b);
            hi[e] = hu(RAW && e % 2 ? __hmul2(h, __float2half2_rn(0.0625f)) : h);
            if constexpr (std::is_same<T, float>::value) {
                const float2 back = __half22float2(h);
                lo[e] = hu(__floats2half2_rn(a - back.x, b - back.y));
            }
        }
        *reinterpret_cast<uint4 *>(high + 2 * i) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        if constexpr (std::is_same<T, float>::value) *reinterpret_cast<uint4 *>(low + 2 * i) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
}
// of a score to the power of two (never 0: a masked score stays -inf), and the logarithm of the row's sum; a row that saw nothing has no weights
__device__ __forceinline__ float2 row_factors(float scale, float up, float lse) {
    return make_float2(fmaxf(fabsf(scale) * 1.4426950408889634f * __int_as_float((254 << 23) - (__float_as_int(up) & 0x7f800000)), FLT_MIN), lse == -INFINITY ? INFINITY : lse * 1.4426950408889634f);
}
// how many positions up to a row's own one see a cell; the row at p sees it if (unsigned) (p - cell) is below (p < 0 are -1: no cell at all)
__device__ __forceinline__ uint32_t reach(const Kv4Attn & A, int cell) { return A.window > 0 && cell >= A.first ? (uint32_t) A.window : 0x80000000u; }
// ---- keys: eight numbers of each block of a cell, as the rows h of an A operand of 16 cells; odd: the cell, whose scales lie behind its even neighbour's ----
template <int D>
__device__ __forceinline__ void key_halves(const uint8_t * row, const uint8_t * scales, int odd, uint32_t (&kf)[D / 32][2][4], int h) {
    constexpr int NB = D / 32;
    uint32_t w[NB], d[NB];
    if constexpr (NB == 4) {
        *reinterpret_cast<uint4 *>(w) = *reinterpret_cast<const uint4 *>(row);
        *reinterpret_cast<uint4 *>(d) = *reinterpret_cast<const uint4 *>(scales);
    } else {
        *reinterpret_cast<uint2 *>(w) = *reinterpret_cast<const uint2 *>(row);
        *reinterpret_cast<uint2 *>(d) = *reinterpret_cast<const uint2 *>(scales);
    }
    const __half2 e = __float2half2_rn(1032.f), o = __float2half2_rn(72.f);        // 1024 + 8, 64 + 8
#pragma unroll
    for (int b = 0; b < NB; b++) {
        const __half2 sc = uh(__byte_perm(d[b], 0u, odd ? 0x3232u : 0x1010u));
        const uint32_t x = w[b], y = w[b] >> 8;
        kf[b][0][h] = hu(__hmul2(__hsub2(uh((x & 0x000f000fu) | 0x64006400u), e), sc));
        kf[b][0][2 + h] = hu(__hmul2(__hsub2(uh((x & 0x00f000f0u) | 0x54005400u), o), sc));
        kf[b][1][h] = hu(__hmul2(__hsub2(uh((y & 0x000f000fu) | 0x64006400u), e), sc));
        kf[b][1][2 + h] = hu(__hmul2(__hsub2(uh((y & 0x00f000f0u) | 0x54005400u), o), sc));
    }
}
// a cell's words as they are, and the blocks' scales
template <int D>
__device__ __forceinline__ void key_words(const uint8_t * row, const uint8_t * scales, int odd, uint32_t (&w)[D / 32], float (&sc)[D / 32]) {
    constexpr int NB = D / 32;
    uint32_t d[NB];
    if constexpr (NB == 4) {
        *reinterpret_cast<uint4 *>(w) = *reinterpret_cast<const uint4 *>(row);
        *reinterpret_cast<uint4 *>(d) = *reinterpret_cast<const uint4 *>(scales);
    } else {
        *reinterpret_cast<uint2 *>(w) = *reinterpret_cast<const uint2 *>(row);
        *reinterpret_cast<uint2 *>(d) = *reinterpret_cast<const uint2 *>(scales);
    }
#pragma unroll
    for (int b = 0; b < NB; b++) sc[b] = __half2float(__ushort_as_half((unsigned short) (odd ? d[b] >> 16 : d[b])));
}
// scores of 32 cells and eight rows: lane: cells 16 m + g, + 8 of rows 2 c, 2 c + 1; q: this lane's part of row g, the low parts `low` bytes further on: these first (what is added to a sum is cut off)
template <int LO, int NB>
__device__ __forceinline__ void scores(const uint32_t (&kf)[2][NB][2][4], const uint8_t * q, size_t low, float (&acc)[2][4]) {
#pragma unroll
    for (int m = 0; m < 2; m++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[m][i] = 0.f;
#pragma unroll
    for (int part = LO - 1; part >= 0; part--)
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const uint4 x = *reinterpret_cast<const uint4 *>(q + part * low + 64 * b);
#pragma unroll
            for (int m = 0; m < 2; m++) {
                mma16816(acc[m], kf[m][b][0], x.x, x.y);
                mma16816(acc[m], kf[m][b][1], x.z, x.w);
            }
        }
}

template <typename T, int D>
__global__ void __launch_bounds__(KW_THREADS, 2) k_kv4_weigh(const __grid_constant__ Kv4Weigh W, const KwSplit X) {
    constexpr bool F32 = std::is_same<T, float>::value;
    constexpr int NB = D / 32, LO = F32 ? 2 : 1;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    KwSmem<D, F32> & S = *reinterpret_cast<KwSmem<D, F32> *>(smem_raw);
    const Kv4Attn & A = W.attn;
    const int tid = threadIdx.x, lane = tid & 31, warp = uniform_warp(), g = lane >> 2, c = lane & 3, hks = A.cache.n_head_kv;
    const int ctas = (int) cluster_size(), rank = (int) cluster_rank();

    pdl_wait();                                             // what attention, or whatever stands in front, has written
    auto length = [&](int s) { return s < A.n_seq ? (int) max((int64_t) 0, min((int64_t) A.kv_len[s], W.ld_sums)) : 0; };
    // items of 256 sequences at a time: where each one's end; the items in front of them
    int at = -1, before = 0, all = 0;
    auto scan = [&](int s0) {
        int x = (length(s0 + tid) + X.cells - 1) / X.cells;
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
        const int base = (item - before - (k > 0 ? S.ends[k - 1] : 0)) * X.cells, len = length(s);

        // ---- the rows that see any of them ----
        const int64_t q0 = A.q_start[s], q1 = A.q_start[s + 1];
        const bool some = q0 >= 0 && q1 > q0 && q1 <= A.n_tokens;
        const int n_all = some ? (int) (q1 - q0) : 0, n_q = min(n_all, A.max_q), p0 = max(A.kv_len[s], 0) - n_all;
        int t_lo = min(n_q, max(0, base - p0)), t_hi = n_q;
        if (A.window > 0 && base >= A.first) t_hi = (int) max((int64_t) t_lo, min((int64_t) n_q, (int64_t) base + X.cells - 1 + A.window - p0));
        const int r_lo = t_lo * A.group, rows = t_hi * A.group - r_lo, blocks = (rows + KW_ROWS - 1) / KW_ROWS, units = hks * blocks;
        const int u0 = (int) ((int64_t) units * rank / ctas), u1 = (int) ((int64_t) units * (rank + 1) / ctas);

        // ---- this warp's cells: page, keys of a kv head ----
        const int cell0 = base + 32 * (warp / X.cuts), in_page = cell0 % KV4_CELLS;
        const int page_at = cell0 / KV4_CELLS;
        int page = -1;
        if (cell0 < len && page_at < A.table_ld) {
            page = A.table[s * A.table_ld + page_at];
            if (page >= A.cache.n_pages) page = -1;
        }
        uint32_t back[2][2];
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
            for (int h = 0; h < 2; h++) back[m][h] = reach(A, cell0 + 16 * m + 8 * h + g);
        uint32_t kf[2][NB][2][4];                           // eights of cells 16 m + g (+ 8): block, half of the eight numbers
        float sum[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
        int held = -1;
        constexpr bool WIDE = std::is_same<T, __nv_bfloat16>::value && D == 128;             // rows by 16 bytes where they lie so (bf16, 2048 x 2048 293 -> 259 us, 64 x 16 000 45 -> 41; heads of 64 2 % slower).  F16 always
        const bool wide = (((uintptr_t) A.q | (uintptr_t) (A.ldq * sizeof(T))) & 15) == 0;
        for (int u = u0; u < u1; u++) {
            const int hk = u / blocks, row0 = r_lo + (u - hk * blocks) * KW_ROWS, n = min(KW_ROWS, r_lo + rows - row0);
            if (held != hk && page >= 0) {
                const uint8_t * chunk = kv4_chunk<D>(A.cache, page, hk), * scales = chunk + 2 * kv4_rows_bytes(D);
#pragma unroll
                for (int m = 0; m < 2; m++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int t = in_page + 16 * m + 8 * h + g;
                        key_halves<D>(chunk + t * (D / 2) + 4 * NB * c, scales + kv4_scale(D, t & ~1, 0), t & 1, kf[m], h);
                    }
                held = hk;
            }
            // the block's rows: four threads to a row, eight numbers each at a time, next to each other
            __syncthreads();
            {
                const int r = tid >> 2, quarter = tid & 3, row = row0 + r, t = row / A.group, head = hk * A.group + row - t * A.group;
                const bool have = r < n;
                constexpr int EACH = D / 4;
                const T * src = (const T *) A.q + (q0 + t) * A.ldq + (int64_t) head * D + 8 * quarter;
                const float lse = have ? W.lse[(q0 + t) * W.ld_lse + head] : -INFINITY;
                float up = 1.f;
                if constexpr (std::is_same<T, __half>::value) {            // as they are
                    const uint32_t turned = A.scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
                    for (int i = 0; i < EACH; i += 8) {
                        uint4 w = make_uint4(0u, 0u, 0u, 0u);
                        if (have) {
                            if (wide) w = *reinterpret_cast<const uint4 *>(src + 4 * i);
                            else {
                                const uint2 x = *reinterpret_cast<const uint2 *>(src + 4 * i), y = *reinterpret_cast<const uint2 *>(src + 4 * i + 4);
                                w = make_uint4(x.x, x.y, y.x, y.y);
                            }
                        }
                        *reinterpret_cast<uint4 *>(&S.q[0][r][16 * quarter + 8 * i]) = make_uint4(w.x ^ turned, w.y ^ turned, w.z ^ turned, w.w ^ turned);
                    }
                } else {
                    float x[EACH];
#pragma unroll
                    for (int i = 0; i < EACH; i += 8) {
                        __align__(16) T w[8];
                        if (WIDE && wide) *reinterpret_cast<uint4 *>(w) = have ? *reinterpret_cast<const uint4 *>(src + 4 * i) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
                        for (int k = 0; k < 8; k += 4) {
                            const float4 v = WIDE && wide ? load4(w + k) : have ? load4(src + 4 * i + k) : make_float4(0.f, 0.f, 0.f, 0.f);
                            x[i + k] = v.x; x[i + k + 1] = v.y; x[i + k + 2] = v.z; x[i + k + 3] = v.w;
                        }
                    }
                    up = row_power<EACH>(x) * (A.scale < 0.f ? -1.f : 1.f);
#pragma unroll
                    for (int i = 0; i < EACH; i += 8) row_store<T, 8>(reinterpret_cast<float(&)[8]>(x[i]), up, &S.q[0][r][16 * quarter + 8 * i], &S.q[LO - 1][r][16 * quarter + 8 * i]);
                }
                if (quarter == 0) {
                    S.row[r] = row_factors(A.scale, up, lse);
                    S.pos[r] = have ? max(p0 + t, -1) : -1;
                }
            }
            __syncthreads();
            const int p_lo = p0 + row0 / A.group, p_hi = p0 + (row0 + n - 1) / A.group;
            if (page < 0 || cell0 > p_hi) continue;
            const bool whole = cell0 + 31 <= p_lo && (A.window <= 0 || p_hi - cell0 < A.window || cell0 + 31 < A.first);
#pragma unroll 1
            for (int j = 16 * (warp % X.cuts); j < n; j += 16 * X.cuts) {      // two tiles of rows at once: one's products beside the other's weights
                float e[2][2][4];
#pragma unroll
                for (int t = 0; t < 2; t++) scores<LO, NB>(kf, &S.q[0][j + 8 * t + g][16 * c], sizeof(S.q[0]), e[t]);
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    const float4 r = *reinterpret_cast<const float4 *>(&S.row[j + 8 * t + 2 * c]);
#pragma unroll
                    for (int m = 0; m < 2; m++)
#pragma unroll
                        for (int i = 0; i < 4; i++) e[t][m][i] = ex2(fmaf(e[t][m][i], i & 1 ? r.z : r.x, i & 1 ? -r.w : -r.y));
                    if (!whole) {
                        const int2 pos = *reinterpret_cast<const int2 *>(&S.pos[j + 8 * t + 2 * c]);
#pragma unroll
                        for (int m = 0; m < 2; m++)
#pragma unroll
                            for (int i = 0; i < 4; i++)
                                if ((uint32_t) ((i & 1 ? pos.y : pos.x) - (cell0 + 16 * m + 8 * (i >> 1) + g)) >= back[m][i >> 1]) e[t][m][i] = 0.f;
                    }
#pragma unroll
                    for (int m = 0; m < 2; m++) {
                        sum[m][0] += e[t][m][0] + e[t][m][1];
                        sum[m][1] += e[t][m][2] + e[t][m][3];
                    }
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
                if (c == 0) S.part[flip][warp % X.cuts * X.cells + 32 * (warp / X.cuts) + 16 * m + 8 * h + g] = x;
            }
        cluster_sync();                                     // (of the item behind the next one's, nobody reads these any more)
        for (int i = rank * X.cells / ctas + tid; i < (rank + 1) * X.cells / ctas; i += KW_THREADS) {
            float x = 0.f;
            for (int r = 0; r < ctas; r++)
                for (int w = 0; w < X.cuts; w++) x += remote(&S.part[flip][w * X.cells + i], r);
            const int64_t j = base + i;
            if (j < len) W.sums[s * W.ld_sums + j] = W.old ? fmaf(W.decay, W.old[s * W.ld_old + j], x) : x;
        }
        flip ^= 1;
    }
}

// ---- few rows ----
// Pages stream through shared memory, by bulk copies: a warp has the keys of a page and a kv head at a time, the next ones on their way, and all of the head's rows.  A unit is as many pages of a
// sequence as give each warp such a turn; a CTA has a contiguous share of all units.  The queries of all heads lie in shared memory while it is at their sequence.
constexpr int KF_WARPS = 16, KF_THREADS = 32 * KF_WARPS;
__host__ __device__ constexpr int kf_bytes(int D) { return kv4_rows_bytes(D) + kv4_scales_bytes(D); }     // of a page's keys
constexpr int KF_STAGES = 2, KF_ROWS = 16;

struct KfSplit { int most_rows; int * abort_flag; };      // rows of a kv head at most
// a sequence: its queries, positions, cells and units
struct KfSeq {
    int64_t q0;
    int n_q, p0, len, units;
};
template <int D> struct __align__(128) KfSmem {
    __align__(128) uint8_t ring[KF_WARPS][KF_STAGES][kf_bytes(D)];
    uint64_t full[KF_WARPS][KF_STAGES];
    float part[2][KF_WARPS][KV4_CELLS];        // of the warps
    int scan[KF_WARPS], begin_s, begin_unit, abort;
    KfSeq begin;
};
// behind it: of all rows (kv head by kv head) and eight more the numbers (F32: high, then low parts), what makes their weights, RAW: where their sums start; the positions of a kv head's
template <typename T, int D> __host__ __device__ constexpr size_t kf_row_bytes() {
    return (std::is_same<T, float>::value ? 2 * (2 * D + 64) : 2 * D + 64 + D / 32 * sizeof(float)) + sizeof(float2);
}

// RAW: 16 bits: the numbers' 4 bits go into the products as they are, as the f16 n * 2^-24 (n * 2^-20 a nibble further up, which meets a 16th of the query), and scales onto the sums of blocks, which
// start from -8 times the query's; making them f16 keys takes twice as many instructions (32 sequences of up to 8192 cells 38 us where this takes 33).  F32 has
// twice the products as it is, and keeps the f16 keys
template <typename T, int D>
__global__ void __launch_bounds__(KF_THREADS, 1) k_kv4_weigh_few(const __grid_constant__ Kv4Weigh W, const __grid_constant__ KfSplit X) {
    constexpr bool F32 = std::is_same<T, float>::value;
    constexpr bool RAW = !F32;
    constexpr int NB = D / 32, LO = F32 ? 2 : 1, STAGES = KF_STAGES, STRIDE = 2 * D + 64;
    extern __shared__ uint8_t smem_raw[];
    KfSmem<D> & S = *reinterpret_cast<KfSmem<D> *>(smem_raw + ((128u - (smem_u32(smem_raw) & 127u)) & 127u));
    const Kv4Attn & A = W.attn;
    const int tid = threadIdx.x, lane = tid & 31, warp = uniform_warp(), g = lane >> 2, c = lane & 3;
    uint8_t * const queries = reinterpret_cast<uint8_t *>(&S + 1);
    const int hks = A.cache.n_head_kv, room = hks * X.most_rows + 8;                // rows
    float2 * const factors = reinterpret_cast<float2 *>(queries + (size_t) room * STRIDE * LO);
    float * const starts = reinterpret_cast<float *>(factors + room);        // RAW: of each row and block
    int * const pos = reinterpret_cast<int *>(starts + (RAW ? room * NB : 0));
    volatile int * cta_abort = &S.abort;
    // pages of a unit; this warp's page of them and its first head (`hks` and more: none)
    const int P = max(1, KF_WARPS / hks), my_page = P > 1 ? warp / hks : 0, my_head = P > 1 ? (my_page < P ? warp % hks : hks) : warp;

    auto seq = [&](int s) {
        KfSeq q{};
        if (s >= A.n_seq) return q;
        const int64_t a = A.q_start[s], b = A.q_start[s + 1];
        const int cells = max(A.kv_len[s], 0);
        q.len = (int) min((int64_t) cells, W.ld_sums);
        q.units = ((q.len + KV4_CELLS - 1) / KV4_CELLS + P - 1) / P;
        q.q0 = a;
        q.p0 = cells;
        if (a >= 0 && b > a && b <= A.n_tokens) {
            q.p0 = cells - (int) (b - a);
            q.n_q = min((int) (b - a), A.max_q);
        }
        return q;
    };
    // ---- the share: units in the order of sequences ----
    if (lane < STAGES) {
        mbar_init(&S.full[warp][lane], 1);
        mbar_fence_init();
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (tid == 0) S.abort = 0;
    pdl_wait();                                             // what attention, or whatever stands in front, has written
    auto upto = [&](int x) {                                // sum over the threads up to this one, all: over all
        int y = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int z = __shfl_up_sync(0xffffffffu, y, o);
            if (lane >= o) y += z;
        }
        __syncthreads();
        if (lane == 31) S.scan[warp] = y;
        __syncthreads();
        return y;
    };
    const KfSeq first = seq(tid);
    int mine = first.units;
    for (int s = tid + KF_THREADS; s < A.n_seq; s += KF_THREADS) mine += seq(s).units;
    int ends = upto(mine);
    long long total = 0;
#pragma unroll
    for (int w = 0; w < KF_WARPS; w++) {
        if (w < warp) ends += S.scan[w];
        total += S.scan[w];
    }
    const int u0 = (int) (total * blockIdx.x / gridDim.x), u1 = (int) (total * (blockIdx.x + 1) / gridDim.x);
    if (u0 == u1) return;
    auto begins = [&](int s, const KfSeq & q, int before) {
        if (u0 >= before && u0 < before + q.units) { S.begin_s = s; S.begin_unit = u0 - before; S.begin = q; }
    };
    if (A.n_seq <= KF_THREADS) begins(tid, first, ends - mine);
    else
        for (int s0 = 0, before = 0; s0 < A.n_seq && before <= u0; s0 += KF_THREADS) {
            const KfSeq q = seq(s0 + tid);
            int x = upto(q.units) - q.units + before;
#pragma unroll
            for (int w = 0; w < KF_WARPS; w++) {
                if (w < warp) x += S.scan[w];
                before += S.scan[w];
            }
            begins(s0 + tid, q, x);
        }
    __syncthreads();

    // ---- this warp's keys on their way: by units and, where there are more heads than warps, heads ----
    uint64_t policy;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    int f_s = S.begin_s, f_unit = S.begin_unit, f_u = u0, f_head = my_head, f_n = 0;
    KfSeq f_q = S.begin;
    int ids = -1, ids0 = 0, ids1 = 0;                       // pages of the units ids0 .. ids1 - 1 of the sequence, one to a lane
    uint32_t none = 0;                                      // stages whose page nobody sees, or that is none
    auto sees = [&](const KfSeq & q, int base) {            // any query any of the page's cells
        return q.n_q > 0 && base <= q.p0 + q.n_q - 1 && (A.window <= 0 || q.p0 - (base + KV4_CELLS - 1) < A.window || base < A.first);
    };
    auto fetch = [&] {
        if (f_u >= u1 || f_head >= hks) return;
        while (f_unit >= f_q.units) {
            f_q = seq(++f_s);
            f_unit = 0;
            ids1 = 0;
        }
        if (f_unit >= ids1) {
            const int at = (f_unit + lane) * P + my_page;
            ids = at < A.table_ld && f_unit + lane < f_q.units && at * KV4_CELLS < f_q.len ? A.table[f_s * A.table_ld + at] : -1;
            ids0 = f_unit;
            ids1 = f_unit + 32;
        }
        int id = __shfl_sync(0xffffffffu, ids, f_unit - ids0);
        if (id >= A.cache.n_pages || !sees(f_q, (f_unit * P + my_page) * KV4_CELLS)) id = -1;
        const int st = f_n % STAGES;
        none = id >= 0 ? none & ~(1u << st) : none | 1u << st;
        if (elect_one()) {
            if (id >= 0) {
                const uint8_t * chunk = kv4_chunk<D>(A.cache, id, f_head);
                mbar_arrive_expect_tx(&S.full[warp][st], kf_bytes(D));
                bulk_g2s(S.ring[warp][st], chunk, kv4_rows_bytes(D), &S.full[warp][st], policy);
                bulk_g2s(S.ring[warp][st] + kv4_rows_bytes(D), chunk + 2 * kv4_rows_bytes(D), kv4_scales_bytes(D), &S.full[warp][st], policy);
            } else mbar_arrive(&S.full[warp][st]);
        }
        __syncwarp();
        f_n++;
        f_head += KF_WARPS;
        if (P > 1 || f_head >= hks) {
            f_head = my_head;
            f_unit++;
            f_u++;
        }
    };
    int s = S.begin_s, unit = S.begin_unit, n = 0;
    bool fresh = true;
    KfSeq q = S.begin;
    for (int u = u0; u < u1; u++, unit++) {
        while (unit >= q.units) {
            q = seq(++s);
            unit = 0;
            fresh = true;
        }
        const int rows = q.n_q * A.group;
        if (fresh) {   // ---- the sequence's queries: four threads to a row ----  (everybody is through with the last one's: behind the barrier of its last unit)
            fresh = false;
            constexpr int EACH = D / 4, ROWS = KF_THREADS / 4;
            for (int i0 = 0; i0 < hks * rows; i0 += ROWS) {
                const int i = i0 + (tid >> 2), quarter = tid & 3, hk = i / rows, r = i - hk * rows, t = r / A.group, head = hk * A.group + r - t * A.group;
                const bool have = i < hks * rows;
                const T * src = (const T *) A.q + (q.q0 + t) * A.ldq + (int64_t) head * D + quarter * EACH;
                float x[EACH];
#pragma unroll
                for (int k = 0; k < EACH; k += 4) {
                    const float4 v = have ? load4(src + k) : make_float4(0.f, 0.f, 0.f, 0.f);
                    x[k] = v.x; x[k + 1] = v.y; x[k + 2] = v.z; x[k + 3] = v.w;
                }
                const float lse = have ? W.lse[(q.q0 + t) * W.ld_lse + head] : -INFINITY;
                if (f_n == 0)                               // the first keys, behind the first queries
                    for (int k = 0; k < STAGES; k++) fetch();
                const float up = row_power<EACH>(x) * (A.scale < 0.f ? -1.f : 1.f);
                float block = 0.f;                          // sum of the block's numbers
                if (RAW) {
#pragma unroll
                    for (int k = 0; k < EACH; k++) block += x[k];
                    if (EACH == 16) block += __shfl_xor_sync(0xffffffffu, block, 1);
                }
                if (!have) continue;
                row_store<T, EACH, RAW>(x, up, queries + (size_t) i * STRIDE + 2 * quarter * EACH, queries + (size_t) (room + i) * STRIDE + 2 * quarter * EACH);
                if (RAW && (EACH == 32 || quarter % 2 == 0)) starts[i * NB + quarter * EACH / 32] = block * (up * (-8.f / 16777216.f));
                if (quarter == 0) {
                    factors[i] = row_factors(A.scale, up, lse);
                    if (RAW) factors[i].x *= 16777216.f;
                    if (i < rows) pos[i] = max(q.p0 + t, -1);
                }
            }
            if (f_n == 0)
                for (int k = 0; k < STAGES; k++) fetch();
            __syncthreads();
        }
        // what the sums are added to, on its way
        const int cells = P * KV4_CELLS;
        float past[2] = {0.f, 0.f};
        if (W.old)
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const int i = k * KF_THREADS + tid;
                const int64_t j = (int64_t) unit * cells + i;
                if (i < cells && j < q.len) past[k] = W.old[s * W.ld_old + j];
            }
        float sum[4][2];
#pragma unroll
        for (int m = 0; m < 4; m++) sum[m][0] = sum[m][1] = 0.f;
        const int base = (unit * P + my_page) * KV4_CELLS;
        for (int hk = my_head; hk < hks; hk += P > 1 ? hks : KF_WARPS, n++) {
            const int st = n % STAGES;
            const bool have = !(none >> st & 1);
            mbar_wait(&S.full[warp][st], (uint32_t) (n / STAGES) & 1, cta_abort, X.abort_flag);
            if (have) {
                const uint8_t * chunk = S.ring[warp][st], * scales = chunk + kv4_rows_bytes(D);
                const int p_lo = q.p0, p_hi = q.p0 + q.n_q - 1;
                const bool whole = base + KV4_CELLS - 1 <= p_lo && (A.window <= 0 || p_hi - base < A.window || base + KV4_CELLS - 1 < A.first);
                if constexpr (RAW) {
#pragma unroll 1
                    for (int j = 0; j < rows; j += 8) {
                        const int i = hk * rows + j;
                        const float2 r0 = factors[i + 2 * c], r1 = factors[i + 2 * c + 1];
                        uint4 qf[NB];
                        float from[NB][2];
#pragma unroll
                        for (int b = 0; b < NB; b++) {
                            qf[b] = *reinterpret_cast<const uint4 *>(queries + (size_t) (i + g) * STRIDE + 64 * b + 16 * c);
                            from[b][0] = starts[(i + 2 * c) * NB + b];
                            from[b][1] = starts[(i + 2 * c + 1) * NB + b];
                        }
                        const bool ra = j + 2 * c < rows, rb = j + 2 * c + 1 < rows;
                        const int pa = whole || !ra ? -1 : pos[j + 2 * c], pb = whole || !rb ? -1 : pos[j + 2 * c + 1];
#pragma unroll
                        for (int m = 0; m < 4; m++) {       // 16 cells at a time
                            uint32_t w[2][NB];
                            float sc[2][NB], e[4];
#pragma unroll
                            for (int h = 0; h < 2; h++) key_words<D>(chunk + (16 * m + 8 * h + g) * (D / 2) + 4 * NB * c, scales + kv4_scale(D, (16 * m + 8 * h + g) & ~1, 0), g & 1, w[h], sc[h]);
#pragma unroll
                            for (int b = 0; b < NB; b++) {
                                const uint32_t x = w[0][b], y = w[1][b], x8 = x >> 8, y8 = y >> 8;
                                const uint32_t a0[4] = {x & 0x000f000fu, y & 0x000f000fu, x & 0x00f000f0u, y & 0x00f000f0u}, a1[4] = {x8 & 0x000f000fu, y8 & 0x000f000fu, x8 & 0x00f000f0u, y8 & 0x00f000f0u};
                                float acc[4] = {from[b][0], from[b][1], from[b][0], from[b][1]};
                                mma16816<true>(acc, a0, qf[b].x, qf[b].y);
                                mma16816<true>(acc, a1, qf[b].z, qf[b].w);
#pragma unroll
                                for (int k = 0; k < 4; k++) e[k] = b == 0 ? acc[k] * sc[k >> 1][b] : fmaf(acc[k], sc[k >> 1][b], e[k]);
                            }
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                const float x = ex2(fmaf(e[k], k & 1 ? r1.x : r0.x, k & 1 ? -r1.y : -r0.y));
                                e[k] = (k & 1 ? rb : ra) ? x : 0.f;
                            }
                            if (!whole)
#pragma unroll
                                for (int k = 0; k < 4; k++) {
                                    const int cell = base + 16 * m + 8 * (k >> 1) + g, p = k & 1 ? pb : pa;
                                    if ((uint32_t) (p - cell) >= reach(A, cell)) e[k] = 0.f;
                                }
                            sum[m][0] += e[0] + e[1];
                            sum[m][1] += e[2] + e[3];
                        }
                    }
                } else
#pragma unroll 1
                for (int m2 = 0; m2 < 2; m2++) {            // 32 cells at a time
                    uint32_t kf[2][NB][2][4];
#pragma unroll
                    for (int m = 0; m < 2; m++)
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const int t = 32 * m2 + 16 * m + 8 * h + g;
                            key_halves<D>(chunk + t * (D / 2) + 4 * NB * c, scales + kv4_scale(D, t & ~1, 0), t & 1, kf[m], h);
                        }
                    float acc2[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
                    auto weights = [&](int j, float (&e)[2][4]) {       // of rows j .. j + 7, from their scores
                        const int i = hk * rows + j;
                        const float2 r0 = factors[i + 2 * c], r1 = factors[i + 2 * c + 1];
#pragma unroll
                        for (int m = 0; m < 2; m++)
#pragma unroll
                            for (int k = 0; k < 4; k++) e[m][k] = ex2(fmaf(e[m][k], k & 1 ? r1.x : r0.x, k & 1 ? -r1.y : -r0.y));
                        if (j + 8 > rows) {                   // rows of nobody's
                            const bool ra = j + 2 * c < rows, rb = j + 2 * c + 1 < rows;
#pragma unroll
                            for (int m = 0; m < 2; m++)
#pragma unroll
                                for (int k = 0; k < 4; k++) e[m][k] = (k & 1 ? rb : ra) ? e[m][k] : 0.f;
                        }
                        if (!whole) {
                            const int pa = j + 2 * c < rows ? pos[j + 2 * c] : -1, pb = j + 2 * c + 1 < rows ? pos[j + 2 * c + 1] : -1;
#pragma unroll
                            for (int m = 0; m < 2; m++)
#pragma unroll
                                for (int k = 0; k < 4; k++) {
                                    const int cell = base + 32 * m2 + 16 * m + 8 * (k >> 1) + g, p = k & 1 ? pb : pa;
                                    if ((uint32_t) (p - cell) >= reach(A, cell)) e[m][k] = 0.f;
                                }
                        }
#pragma unroll
                        for (int m = 0; m < 2; m++) {
                            acc2[m][0] += e[m][0] + e[m][1];
                            acc2[m][1] += e[m][2] + e[m][3];
                        }
                    };
                    const uint8_t * const q_at = queries + (size_t) (hk * rows + g) * STRIDE + 16 * c;
                    int j = 0;
#pragma unroll 1
                    for (; j + 8 < rows; j += 16) {           // two tiles of rows at once: one's products beside the other's weights
                        float e0[2][4], e1[2][4];
                        scores<LO, NB>(kf, q_at + (size_t) j * STRIDE, (size_t) room * STRIDE, e0);
                        scores<LO, NB>(kf, q_at + (size_t) (j + 8) * STRIDE, (size_t) room * STRIDE, e1);
                        weights(j, e0);
                        weights(j + 8, e1);
                    }
                    if (j < rows) {
                        float e0[2][4];
                        scores<LO, NB>(kf, q_at + (size_t) j * STRIDE, (size_t) room * STRIDE, e0);
                        weights(j, e0);
                    }
#pragma unroll
                    for (int m = 0; m < 2; m++)
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            if (m2 == 0) sum[m][h] += acc2[m][h];
                            else sum[2 + m][h] += acc2[m][h];
                        }
                }
            }
            __syncwarp();
            fetch();
        }
        // ---- the warps' sums: of a page those of its kv heads, in their order ----
        const int flip = u & 1;
        if (my_head < hks)
#pragma unroll
            for (int m = 0; m < 4; m++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    float x = sum[m][h];
                    x += __shfl_xor_sync(0xffffffffu, x, 1);
                    x += __shfl_xor_sync(0xffffffffu, x, 2);
                    if (c == 0) S.part[flip][warp][16 * m + 8 * h + g] = x;
                }
        __syncthreads();                                    // (of the unit behind the next one's, nobody reads these any more)
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const int i = k * KF_THREADS + tid, page = i / KV4_CELLS, w0 = P > 1 ? page * hks : 0, w1 = P > 1 ? w0 + hks : min(KF_WARPS, hks);
            const int64_t j = (int64_t) unit * cells + i;
            if (i >= cells || j >= q.len) continue;
            float x = 0.f;
            for (int w = w0; w < w1; w++) x += S.part[flip][w][i % KV4_CELLS];
            W.sums[s * W.ld_sums + j] = fmaf(W.decay, past[k], x);
        }
    }
}

template <typename T, int D>
int weigh_launch(const Kv4Weigh & w, cudaStream_t st) {
    const int hks = w.attn.cache.n_head_kv;
    const int64_t rows = std::min<int64_t>(w.attn.max_q, w.attn.n_tokens) * w.attn.group;
    // Few rows: those of all heads lie in an SM's shared memory, beside the keys that stream through it; keys are read once, where the other kernel's CTAs each load and convert 64 rows whatever there are.
    // bf16, 32 query heads of 8, D = 128, 20 sequences of 100 .. 4000 cells: 4 rows to a kv head 16 us against 27, 16 rows 23 against 28; 32 sequences, 20 rows 33 against 35.  One kv head, 5000 cells: 32
    // rows 10.9 against 6.9
    if (rows <= KF_ROWS) {
        const size_t few = sizeof(KfSmem<D>) + 128 + (size_t) (hks * rows + 8) * kf_row_bytes<T, D>() + 4 * (size_t) rows;
        if (few <= 232448) {
            static FuncAttrCache cache;
            const cudaError_t e = ensure_dyn_smem(cache, (const void *) k_kv4_weigh_few<T, D>, 232448, true);
            if (e != cudaSuccess) return (int) e;
            return (int) launch_clusters(k_kv4_weigh_few<T, D>, sm_count(), 1, KF_THREADS, few, true, st, w, KfSplit{(int) rows, abort_flag()});
        }
    }
    constexpr size_t smem = sizeof(KwSmem<D, std::is_same<T, float>::value>);
    static FuncAttrCache cache;
    cudaError_t e = ensure_dyn_smem(cache, (const void *) k_kv4_weigh<T, D>, smem, false);
    if (e != cudaSuccess) return (int) e;
    const int64_t units = hks * ((rows + KW_ROWS - 1) / KW_ROWS);
    // How items are cut, by what a launch takes, in us: an item 6, a unit 1.2 to load and convert and 2 for its products, where two CTAs share an SM 0.8 + 2 for each; items behind those at once wait.
    // Measured (rows by 8 bytes), bf16, 32 query heads of 8, D = 128: 64 queries x 16 000 cells 1 CTA 112, 4 CTAs 45, 8 62, 4 with warps in pairs 62; 100 x 1000 8 CTAs 29, in pairs 23; 2048 x 2048 411 and 293.
    const int64_t cells = std::min<int64_t>(w.ld_sums, (int64_t) w.attn.table_ld * KV4_CELLS);
    int ctas = 1, cuts = 1;
    double best = INFINITY;
    for (int n = 1; n <= 8; n *= 2)
        for (int k = 1; k <= 4; k *= 2) {
            const double items = (double) w.attn.n_seq * ((cells + KW_CELLS / k - 1) / (KW_CELLS / k)), rounds = std::ceil(items / (2 * clusters_at_once(n, sm_count()))), per_sm = std::min(2.0, items * n / sm_count());
            const double t = rounds * ((units + n - 1) / n * std::max(1.2 + 2.0 / k, per_sm * (0.8 + 2.0 / k)) + 6);
            if (t < best) { best = t; ctas = n; cuts = k; }
        }
    return (int) launch_clusters(k_kv4_weigh<T, D>, 2 * clusters_at_once(ctas, sm_count()), ctas, KW_THREADS, smem, true, st, w, KwSplit{KW_CELLS / cuts, cuts});
}

}  // namespace

int launch_kv4_weigh(const Kv4Weigh & w, int D, int type, cudaStream_t st) {
    if (D == 128) return type == PB200_TYPE_F32 ? weigh_launch<float, 128>(w, st) : type == PB200_TYPE_F16 ? weigh_launch<__half, 128>(w, st) : weigh_launch<__nv_bfloat16, 128>(w, st);
    return type == PB200_TYPE_F32 ? weigh_launch<float, 64>(w, st) : type == PB200_TYPE_F16 ? weigh_launch<__half, 64>(w, st) : weigh_launch<__nv_bfloat16, 64>(w, st);
}

}  // namespace pb
