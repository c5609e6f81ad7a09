// prima.cpp_b200/csrc/kv4_attn.cuh — what the attention kernels over the 4-bit cache share: which pages a sequence's queries see, and in what order.
#pragma once
#include "kv4.cuh"
#include "tc.cuh"

namespace pb {

constexpr int KV4_MAX_CTAS = 152;      // of a launch: the workspace has parts by CTA and warp
constexpr int KV4_SLOTS = 2 * KV4_MAX_CTAS;   // and by piece of a cut item: these are 9 / 5 of the CTAs at most (F32's have half of their rows: the other half of two is a CTA's)
constexpr int KV4_COUNTERS = 16384;    // in front of them

// A sequence: its queries' rows, and the pages that any of them sees: the first `keep`, then those from page `from` on.  At least one page, so that rows which see
// nothing are written.  All numbers come from device memory and are taken for what they may be: rows beyond the arrays, negative lengths, short tables.
struct Kv4Seq {
    int64_t q0;                // first row
    int n_q, p0;               // queries; position of the first
    int pages, keep, from;
    int n_rows;                // queries x heads of a group
    __device__ __forceinline__ int items(int n_head_kv, int tile) const { return n_q > 0 ? n_head_kv * ((n_rows + tile - 1) / tile) : 0; }
    __device__ __forceinline__ int units(int n_head_kv, int tile) const { return items(n_head_kv, tile) * pages; }
};
// the pages that queries at the positions lo .. hi see
__device__ __forceinline__ void kv4_pages(const Kv4Attn & A, int lo, int hi, Kv4Seq & q) {
    q.pages = 1;
    q.keep = q.from = 0;
    if (hi < 0) return;
    const int ld = (int) (A.table_ld < 0x1ffffff ? A.table_ld : 0x1ffffff);   // cells have 31 bits
    const int last = min(hi / KV4_CELLS, ld - 1);
    if (A.window > 0 && lo >= A.window) {
        q.from = (lo - A.window + 1) / KV4_CELLS;
        q.keep = min(min(A.first / KV4_CELLS + (A.first % KV4_CELLS != 0), q.from), last + 1);
    }
    q.pages = max(1, q.keep + max(0, last + 1 - q.from));
}
// many: sequences with more than most_rows rows, otherwise the others
template <bool X>
__device__ __forceinline__ Kv4Seq kv4_seq(const Kv4Attn & A, int s, int most_rows, bool many) {
    Kv4Seq q{};
    if (s >= A.n_seq) return q;
    int s0 = s, s1 = s + 1;
    if (X && A.x.all) {
        s0 = A.x.group_start[s];
        s1 = A.x.group_start[s + 1];
        if (s0 < 0 || s1 <= s0 || s1 > A.x.n_seq) return q;
    }
    const long long a = A.q_start[s0], b = A.q_start[s1], cells = A.kv_len[s];     // (all on their way)
    if (a < 0 || b <= a || b > A.n_tokens) return q;
    const int all = (int) (b - a), n = min(all, A.max_q);
    if (((long long) n * A.group > most_rows) != many) return q;
    q.q0 = a;
    q.n_q = n;
    q.n_rows = n * A.group;
    const int len = max((int) cells, 0);
    if (X && A.x.all) {
        q.p0 = len - 1;
        kv4_pages(A, q.p0, q.p0, q);
        return q;
    }
    q.p0 = len - all;
    kv4_pages(A, q.p0, q.p0 + n - 1, q);
    return q;
}
// position of a sequence's query
template <bool X> __device__ __forceinline__ int kv4_pos(const Kv4Attn & A, const Kv4Seq & q, int t) { return X && A.x.all ? q.p0 : q.p0 + t; }
// the i-th of its pages: which one of the sequence, and its number in the pool (-1: none)
__device__ __forceinline__ int kv4_page_index(const Kv4Seq & q, int i) { return i < q.keep ? i : i - q.keep + q.from; }
template <bool X>
__device__ __forceinline__ int kv4_page(const Kv4Attn & A, const Kv4Seq & q, int s, int i) {
    const int at = kv4_page_index(q, i);
    if ((X && A.x.all ? q.p0 < 0 : q.p0 + q.n_q <= 0) || at >= A.table_ld) return -1;
    const int id = A.table[s * A.table_ld + at];
    return id >= 0 && id < A.cache.n_pages ? id : -1;
}

// of a part with maximum m and sum l of weights, where all parts' maximum is top (a row that is no number has no maximum)
__device__ __forceinline__ float part_factor(float m, float l, float top) { return m == -INFINITY ? (l == l ? 0.f : 1.f) : ex2(m - top); }

// What becomes of a row's sum of values x, times 2^-m and with l the sum of its weights: own * x + other * from, into `to` or, as a part, into `put`
struct Kv4Row { float own, other; const float * from; float * put; };
template <int D>
__device__ __forceinline__ Kv4Row kv4_row(const Kv4Attn & A, int s, int64_t token, int head, float m, float l, bool writes) {
    const int64_t at = token * A.n_head + head;
    Kv4Row r{0.f, 0.f, nullptr, nullptr};
    if (A.x.part == KV4_PUT) {
        if (writes) A.x.ml[at] = make_float2(m, l);
        r.own = 1.f;
        r.put = A.x.o + at * D;
        return r;
    }
    float all = l, top = m, f = 1.f;
    if (A.x.part == KV4_FOLD && s >= A.x.group_start[0] && s < A.x.group_start[A.x.n_group]) {
        const float2 p = A.x.ml[at];
        top = fmaxf(m, p.x);
        f = part_factor(m, l, top);
        r.other = part_factor(p.x, p.y, top);
        r.from = A.x.o + at * D;
        all = l * f + p.y * r.other;
    }
    const float inv = all == 0.f ? 0.f : 1.f / all;
    r.own = f * inv;
    r.other *= inv;
    if (writes && A.x.lse) A.x.lse[token * A.x.ld_lse + head] = all == 0.f ? -INFINITY : (top + log2f(all)) * 0.6931471805599453f;
    return r;
}
__device__ __forceinline__ float4 kv4_mix(const Kv4Row & r, float4 x, int d) {      // numbers d .. d + 3
    float4 y = make_float4(x.x * r.own, x.y * r.own, x.z * r.own, x.w * r.own);
    if (r.from) {
        const float4 z = *reinterpret_cast<const float4 *>(r.from + d);
        y.x = fmaf(z.x, r.other, y.x); y.y = fmaf(z.y, r.other, y.y); y.z = fmaf(z.z, r.other, y.z); y.w = fmaf(z.w, r.other, y.w);
    }
    return y;
}

__device__ __forceinline__ void tmem_alloc(uint32_t * at, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(at)), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t columns) { asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns) : "memory"); }

struct KrWork { int most_rows; int * counters; void * parts; int * abort_flag; };
size_t kv4_rows_workspace(int D);
int launch_kv4_attn_rows(const Kv4Attn & a, int D, int type, int most_rows, int * counters, void * parts, cudaStream_t st, bool ext);
size_t kv4_prompt_workspace(int D);
int launch_kv4_attn_prompt(const Kv4Attn & a, int D, int type, int most_rows, int * tickets, void * parts, cudaStream_t st, bool ext, int & launches);

}  // namespace pb
