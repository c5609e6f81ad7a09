// prima.cpp_b200/csrc/kv4.cuh — the cache of 4-bit keys and values in pages: where its bits lie, and how numbers become them.
//
// A page holds 64 cells; per layer and kv head it is a chunk: 64 key rows of D / 2 bytes, 64 value rows, 64 * D / 32 scales (f16) of the keys, as many of
// the values.  A number is (n - 8) * scale: n its 4 bits, scale that of its block of 32 numbers of the row.  Scales have 8 significant bits, so that a number
// (4 bits more) is an f16 exactly: tensor cores take it as it is, and what comes out does not depend on which kernel read it.
//
// The order of the bits is that in which the threads of an m16n8k16 product hold its B operand (thread 4 g + c: column g, entries 2c, 2c+1, 2c+8, 2c+9), so that
// a thread's part of a row is one load:
//   keys    row t; 32-bit word c * NB + b (c = d / 8 % 4, b = d / 32) has the numbers 32 b + 8 c + e, e = 0 .. 7, number e at bit 4 * (e / 2) + 16 * (e % 2):
//           two of them sit in the halves of a register after one shift and mask.  A thread reads its NB words (all blocks) of a cell at once.
//   values  row r = t - t % 8 + t % 8 / 2 + 4 * (t % 2); 16-bit word (g ^ 4 * (r / 2 % 2)) * NB + b (g = d / 4 % 8) has the numbers 32 b + 4 g + i, at bit 4 i.  Of the
//           eight cells of a column block, threads 4 g + c read cells 2c (rows 0 .. 3), then 2c+1 (rows 4 .. 7): the order of rows and words spreads both over all banks.
//   scales  entry (t / 2 * NB + b) * 2 + t % 2: of two neighbouring cells together
// Rows are whole bytes of one cell: cells are written and copied without touching others.
#pragma once
#include <cuda_bf16.h>

#include "launch.h"

namespace pb {

constexpr int KV4_CELLS = 64;
constexpr float KV4_MOST = 21760.f;   // 8 * the largest scale: 16 scales and 24 scales are f16 numbers, too

__host__ __device__ constexpr int kv4_rows_bytes(int D) { return KV4_CELLS * D / 2; }
__host__ __device__ constexpr int kv4_scales_bytes(int D) { return KV4_CELLS * D / 16; }
__host__ __device__ constexpr int kv4_chunk_bytes(int D) { return 2 * (kv4_rows_bytes(D) + kv4_scales_bytes(D)); }
__host__ __device__ constexpr bool kv4_dim_ok(int D) { return D == 64 || D == 128; }

__host__ __device__ constexpr int kv4_v_row(int t) { return (t & ~7) | ((t & 7) >> 1) | ((t & 1) << 2); }
// byte of 32-bit word (c, b) of a key row, of 16-bit word (g, b) of a value row, of a scale in its part
__host__ __device__ constexpr int kv4_k_word(int D, int t, int c, int b) { return t * (D / 2) + 4 * (c * (D / 32) + b); }
__host__ __device__ constexpr int kv4_v_word(int D, int t, int g, int b) {
    return kv4_v_row(t) * (D / 2) + 2 * ((g ^ (4 * ((kv4_v_row(t) >> 1) & 1))) * (D / 32) + b);
}
__host__ __device__ constexpr int kv4_scale(int D, int t, int b) { return 2 * (((t >> 1) * (D / 32) + b) * 2 + (t & 1)); }

struct Kv4 {   // one layer of a cache, as kernels take it
    uint8_t * base;        // chunk of (page 0, kv head 0)
    int64_t page_stride;   // bytes
    int64_t n_pages;
    int n_head_kv;
};
template <int D>
__device__ __forceinline__ uint8_t * kv4_chunk(const Kv4 & c, int64_t page, int head) {
    return c.base + page * c.page_stride + (int64_t) head * kv4_chunk_bytes(D);
}

// A block's scale from its number of largest magnitude: bf16 rounds to the 8 significant bits
__device__ __forceinline__ float kv4_scale_of(float most) { return __half2float(__float2half_rn(__bfloat162float(__float2bfloat16_rn(most * -0.125f)))); }
// rint(x / scale) + 8 within 0 .. 15, by the reciprocal of the scale (0: of a scale of 0): that product is within 2^-22 of the quotient (of up to 8.03), and only next to a half is the quotient
// itself needed.  Sums with 1.5 * 2^23 round like rint, and hold the number in their last bits: conversions take eight times as long
__device__ __forceinline__ void kv4_bits_of(const float (&x)[4], float scale, float inv, uint32_t (&m)[4]) {
    float n[4];
    bool near = false;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float y = x[i] * inv;
        n[i] = __fadd_rn(y, 12582912.f) - 12582912.f;
        near |= fabsf(fabsf(y - n[i]) - 0.5f) < 4e-6f;
    }
    if (near)
#pragma unroll
        for (int i = 0; i < 4; i++) n[i] = rintf(__fdiv_rn(x[i], scale));
#pragma unroll
    for (int i = 0; i < 4; i++) m[i] = __float_as_uint(__fadd_rn(fminf(fmaxf(n[i], -8.f), 7.f), 12582920.f)) & 15u;
}
// the cache holds numbers only: a value that is none would reach rows that do not see its cell (0 * NaN)
__device__ __forceinline__ float kv4_finite(float x) { return x != x ? 0.f : fminf(fmaxf(x, -KV4_MOST), KV4_MOST); }

__device__ __forceinline__ float4 load4(const float * p) { return *reinterpret_cast<const float4 *>(p); }
__device__ __forceinline__ float4 load4(const __half * p) {
    const uint2 w = *reinterpret_cast<const uint2 *>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&w.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&w.y));
    return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ float4 load4(const __nv_bfloat16 * p) {
    const uint2 w = *reinterpret_cast<const uint2 *>(p);
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
}
__device__ __forceinline__ void store4(float * p, float4 v) { *reinterpret_cast<float4 *>(p) = v; }
__device__ __forceinline__ void store4(__half * p, float4 v) {
    const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
    *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
}
__device__ __forceinline__ void store4(__nv_bfloat16 * p, float4 v) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
}

// ---- launchers; type: PB200_TYPE_F32 / F16 / BF16 of q, k, v and out ----
struct Kv4Rope {           // frequencies of the pairs in 64 bits: an angle of position 100000 has no digits left in 32
    double w[64];
    int n_dims, mode;      // 0: neighbouring pairs, 2: halves
    float mscale;
    const float * freq_factors;
};
int launch_kv4_append(const Kv4 & cache, int D, int type, const void * q, int64_t ldq, void * q_out, int64_t ldqo, const void * k, int64_t ldk, const void * v, int64_t ldv,
                      int64_t n_tokens, int n_head, const int64_t * cells, const int32_t * pos, const float * q_norm, const float * k_norm, float eps, const Kv4Rope & rope,
                      cudaStream_t st);
int launch_kv4_load(const Kv4 & cache, int D, int type, const int64_t * cells, int64_t n, void * k, int64_t ldk, void * v, int64_t ldv, cudaStream_t st);
int launch_kv4_copy_pages(uint8_t * pages, int64_t page_bytes, const int32_t * src, const int32_t * dst, int n, cudaStream_t st);   // src, dst: host
int launch_kv4_compact(uint8_t * pages, int64_t n_pages, int rows, int D, int n_seq, const int32_t * from, int64_t ld_from, const int32_t * to, int64_t ld_to,
                       const int32_t * index, int64_t ld_index, const int32_t * count, int most, cudaStream_t st);   // rows: chunks of a page
// What attention may do besides (kernels with X): rows' logarithms; prefixes that groups of sequences have in common
struct Kv4Ext {
    float * lse; int64_t ld_lse;          // of each query and head; NULL: not wanted
    int mode;
    const int32_t * group_start;          // the groups' first sequences
    const int32_t * prefix_len, * prefix_table;
    int64_t prefix_ld;
    int n_group, n_own, room;             // groups, sequences; cells that a prefix has at most: what its table has room for, in 30 bits
    int64_t least;                        // what has to be saved for prefixes to be by themselves: pages x kv heads x tiles of eight rows, times 16
    int few;                              // sequences with more rows than this walk the prefix whatever the others do (0: there are none)
    int of_seq, of_tile, rows, log_tile;  // of that, a page of a prefix costs a sequence that walks it, with so many rows, and a tile of 2^log_tile rows in the prompts' kernel
    float * o; float4 * ml;               // parts of rows [token][head]: sums [D]; reference, sum of weights, and the mark of the call
    int * sync;                           // calls that have ended, CTAs of a call's last kernel that have
};
// SHARED: a sequence's cells are the prefix's pages and its own behind them, or, where that is much work for the group, its own alone: sums and what belongs to them go into o and ml.  FRONT, behind
// it: a group is a sequence whose queries, those of all its sequences, see all cells of the prefix; to what a sequence left its part of this is added
enum { KV4_PLAIN = 0, KV4_SHARED = 1, KV4_FRONT = 2 };
struct Kv4Attn {
    Kv4 cache;
    const void * q; int64_t ldq;
    void * out; int64_t ldo;
    int n_head, group, n_seq;
    const int32_t * q_start; const int32_t * kv_len; const int32_t * table;
    int64_t table_ld;
    int64_t n_tokens;
    int max_q, window, first;
    float scale;
    Kv4Ext x;
};
// A sequence with up to so many rows (queries x heads of a group) goes to the kernel of few rows, which walks its pages once for every eight of them; the other one has tiles of 128 and
// 256 rows whatever there are.  us, 32 heads over 8, few rows / prompt: bf16, 8 sequences of 4096 cells, 32 rows 48 / 66, 48 60 / 66, 56 69 / 63; 64 of 1000, 32 rows 86 / 113, 48 111 / 113,
// 64 141 / 114; f16, 8 of 4096, 40 rows 57 / 61, 48 65 / 61; 64 of 1000, 40 rows 104 / 111, 48 122 / 111; 4 of 500, 48 rows 25 / 30; F32, 8 of 4096, 20 rows 54 / 68, 32 70 / 69, 40 77 / 69;
// 64 of 1000, 20 rows 107 / 130, 32 135 / 131, 40 154 / 132; 4 of 500, 32 rows 20 / 32.
constexpr int KV4_FEW_ROWS = 48, KV4_FEW_ROWS_F32 = 32;
size_t kv4_attn_workspace(int D);
int launch_kv4_attn(const Kv4Attn & a, int D, int type, void * ws, cudaStream_t st, int & launches);   // launches: kernels, added up
struct Kv4Groups { int n; const int32_t * start; const int32_t * kv_len; const int32_t * table; int64_t table_ld; };
size_t kv4_attn_shared_workspace(int64_t rows, int D);
int launch_kv4_attn_shared(const Kv4Attn & a, const Kv4Groups & g, int D, int type, void * ws, cudaStream_t st, int & launches);
struct Kv4Weigh {
    Kv4Attn attn;
    const float * lse; int64_t ld_lse;
    float decay;
    const float * old; int64_t ld_old;    // NULL: nothing
    float * sums; int64_t ld_sums;
};
int launch_kv4_weigh(const Kv4Weigh & w, int D, int type, cudaStream_t st);

}  // namespace pb
