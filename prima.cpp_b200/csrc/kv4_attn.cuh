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
    // with prefixes there are no windows: KV4_SHARED has in `keep` the pages of the prefix that come first (a query stands 64 * keep further on), in `from` 64 times the group and the cells that
    // the last of them has not; -1 where the prefix is by itself
    __device__ __forceinline__ int items(int n_head_kv, int tile) const { return n_q > 0 ? n_head_kv * ((n_rows + tile - 1) / tile) : 0; }
    __device__ __forceinline__ int units(int n_head_kv, int tile) const { return items(n_head_kv, tile) * pages; }
};
// the pages that queries at the positions lo .. hi see, of a table with ld pages to a row
__device__ __forceinline__ void kv4_pages(const Kv4Attn & A, int64_t table_ld, int lo, int hi, Kv4Seq & q) {
    q.pages = 1;
    q.keep = q.from = 0;
    if (hi < 0) return;
    const int ld = (int) (table_ld < 0x1ffffff ? table_ld : 0x1ffffff);   // cells have 31 bits
    const int last = min(hi / KV4_CELLS, ld - 1);
    if (A.window > 0 && lo >= A.window) {
        q.from = (lo - A.window + 1) / KV4_CELLS;
        q.keep = min(min(A.first / KV4_CELLS + (A.first % KV4_CELLS != 0), q.from), last + 1);
    }
    q.pages = max(1, q.keep + max(0, last + 1 - q.from));
}
template <bool X> __device__ __forceinline__ bool kv4_shared(const Kv4Attn & A) { return X && A.x.mode == KV4_SHARED; }
template <bool X>
__device__ __forceinline__ void kv4_span(const Kv4Attn & A, int lo, int hi, Kv4Seq & q) {
    if (kv4_shared<X>(A)) {
        const int front = q.keep, from = q.from, own = hi - KV4_CELLS * front;
        kv4_pages(A, A.table_ld, own, own, q);
        q.pages = front + (own < 0 && front > 0 ? 0 : q.pages);
        q.keep = front;
        q.from = from;
    } else kv4_pages(A, X && A.x.mode == KV4_FRONT ? A.x.prefix_ld : A.table_ld, lo, hi, q);
}
// what n sequences save of a page if their prefix is by itself
__host__ __device__ __forceinline__ int64_t kv4_saved(const Kv4Ext & x, int64_t n) { return n * x.of_seq - ((n * x.rows - 1 >> x.log_tile) + 1) * x.of_tile; }
// cells of group g's prefix (as many as its table has room for: pages are counted in 31 bits by what tables have), and whether it is by itself: where that saves the group something, and all groups
// enough for the launch, up to KV4_FEW_GROUPS of them; of more, the group's times their number
constexpr int KV4_FEW_GROUPS = 8;
__device__ __forceinline__ int kv4_prefix(const Kv4Attn & A, int g, bool & apart) {
    auto cells = [&](int i) { return min(max(A.x.prefix_len[i], 0), A.x.room); };
    auto saved = [&](int i) {
        const int64_t of_page = kv4_saved(A.x, min(max(A.x.group_start[i + 1], 0), A.x.n_own) - min(max(A.x.group_start[i], 0), A.x.n_own));
        return of_page > 0 ? of_page * ((cells(i) + KV4_CELLS - 1) / KV4_CELLS) : 0;
    };
    const int64_t own = saved(g);
    int64_t all = 0;
    if (A.x.n_group <= KV4_FEW_GROUPS)
#pragma unroll 1
        for (int i = 0; i < A.x.n_group; i++) all += saved(i);
    else all = own * A.x.n_group;
    apart = own > 0 && all >= A.x.least;
    return cells(g);
}
// KV4_SHARED: `keep` and `from` of a sequence, of many rows or not.  A call, not code in its place: kernels have it in many, and what they are short of is the time to fetch code (a token behind 1000 cells 16 -> 14 us)
static __device__ __noinline__ int2 kv4_in_front(const Kv4Attn & A, int s, bool many) {
    const int n = A.x.n_group;
    if (s < A.x.group_start[0] || s >= A.x.group_start[n]) return make_int2(0, 0);
    int g = 0, end = n;                        // group_start[g] <= s < group_start[end]
    while (end - g > 1) {
        const int mid = (g + end) / 2;
        if (A.x.group_start[mid] <= s) g = mid;
        else end = mid;
    }
    bool apart;
    const int cells = kv4_prefix(A, g, apart), pages = (cells + KV4_CELLS - 1) / KV4_CELLS;
    return apart && !many ? make_int2(0, -1) : make_int2(pages, KV4_CELLS * g + (KV4_CELLS * pages - cells));
}
// position of query t of a sequence
template <bool X> __device__ __forceinline__ int kv4_pos(const Kv4Attn & A, const Kv4Seq & q, int t) {
    if (X && A.x.mode == KV4_FRONT) return q.p0;
    return kv4_shared<X>(A) ? max(q.p0 + t, KV4_CELLS * q.keep - 1) : q.p0 + t;
}
// KV4_FRONT: all tokens t0 .. t1 of a group are of one sequence that walks the prefix itself: rows that nothing was left of
static __device__ __noinline__ bool kv4_walks(const Kv4Attn & A, int g, int64_t t0, int64_t t1) {
    int s = max(A.x.group_start[g], 0), end = min(A.x.group_start[g + 1], A.x.n_own);        // q_start[s] <= t0 < q_start[end]
    while (end - s > 1) {
        const int mid = (s + end) / 2;
        if (A.q_start[mid] <= t0) s = mid;
        else end = mid;
    }
    const int64_t a = A.q_start[s], b = A.q_start[s + 1];
    return a <= t0 && t1 < b && min(b - a, (int64_t) A.max_q) * A.group > A.x.few;
}
// many: sequences with more than most_rows rows, otherwise the others
template <bool X>
__device__ __forceinline__ Kv4Seq kv4_seq(const Kv4Attn & A, int s, int most_rows, bool many) {
    Kv4Seq q{};
    if (s >= A.n_seq) return q;
    const bool front = X && A.x.mode == KV4_FRONT;
    int s0 = s, s1 = s + 1, prefix = 0;
    if (front) {
        s0 = max(A.x.group_start[s], 0);
        s1 = min(A.x.group_start[s + 1], A.x.n_own);
        bool apart;
        prefix = kv4_prefix(A, s, apart);
        if (!apart || s1 <= s0) return q;
    }
    long long a = A.q_start[s0], b = A.q_start[s1], cells = front ? prefix : A.kv_len[s];           // (all on their way)
    if (front) {                               // rows of sequences that are none have no marks: what counts is that those of the others are among these
        a = max(a, 0ll);
        b = min(b, (long long) A.n_tokens);
    }
    if (a < 0 || b <= a || b > A.n_tokens) return q;
    const int all = (int) (b - a), n = front ? all : min(all, A.max_q);
    if (((long long) n * A.group > most_rows) != many) return q;
    q.q0 = a;
    q.n_q = n;
    q.n_rows = n * A.group;
    const int len = max((int) cells, 0);
    q.p0 = front ? len - 1 : len - all;
    if (kv4_shared<X>(A)) {
        const int2 front = kv4_in_front(A, s, many);
        q.keep = front.x;
        q.from = front.y;
        q.p0 = min(len, 1 << 30) - all + KV4_CELLS * q.keep;
    }
    kv4_span<X>(A, kv4_pos<X>(A, q, 0), kv4_pos<X>(A, q, n - 1), q);
    return q;
}
// the i-th of its pages: which one of the sequence, and its number in the pool (-1: none)
template <bool X> __device__ __forceinline__ int kv4_page_index(const Kv4Attn & A, const Kv4Seq & q, int i) { return kv4_shared<X>(A) || i < q.keep ? i : i - q.keep + q.from; }
template <bool X>
__device__ __forceinline__ int kv4_page(const Kv4Attn & A, const Kv4Seq & q, int s, int i) {
    int at = kv4_page_index<X>(A, q, i), id, own = q.p0 + q.n_q;           // (own cells, if it is more than 0)
    if (X && A.x.mode == KV4_FRONT) {
        if (q.p0 < 0 || at >= A.x.prefix_ld) return -1;
        id = A.x.prefix_table[s * A.x.prefix_ld + at];
    } else if (kv4_shared<X>(A) && at < q.keep) {
        if (at >= A.x.prefix_ld) return -1;
        id = A.x.prefix_table[q.from / KV4_CELLS * A.x.prefix_ld + at];
    } else {
        if (kv4_shared<X>(A)) {
            at -= q.keep;
            own -= KV4_CELLS * q.keep;
        }
        if (own <= 0 || at >= A.table_ld) return -1;
        id = A.table[s * A.table_ld + at];
    }
    return id >= 0 && id < A.cache.n_pages ? id : -1;
}
// cells behind the end of a prefix, in its last page: [x, y)
template <bool X> __device__ __forceinline__ int2 kv4_hole(const Kv4Attn & A, const Kv4Seq & q) {
    return kv4_shared<X>(A) && q.keep > 0 ? make_int2(KV4_CELLS * q.keep - q.from % KV4_CELLS, KV4_CELLS * q.keep) : make_int2(0, 0);
}
template <bool X> __device__ __forceinline__ bool kv4_in_hole(int2 hole, int cell) { return X && cell >= hole.x && cell < hole.y; }
template <bool X> __device__ __forceinline__ bool kv4_has_hole(int2 hole, int base) { return X && base < hole.y && base + KV4_CELLS > hole.x; }      // a page from cell `base` on

// of a part with maximum m and sum l of weights, where all parts' maximum is top (a row that is no number has no maximum)
__device__ __forceinline__ float part_factor(float m, float l, float top) { return m == -INFINITY ? (l == l ? 0.f : 1.f) : ex2(m - top); }

// What becomes of a row's sum of values x, times 2^-m and with l the sum of its weights: own * x + other * from, or, as a part, x goes to `put`; skip: nothing (the row is nobody's)
struct Kv4Row { float own, other; const float * from; float * put; bool skip; };
template <int D>
__device__ __forceinline__ Kv4Row kv4_row(const Kv4Attn & A, const Kv4Seq & q, int64_t token, int head, float m, float l, bool writes) {
    const int64_t at = token * A.n_head + head;
    Kv4Row r{0.f, 0.f, nullptr, nullptr, false};
    float all = l, top = m, f = 1.f;
    if (A.x.mode == KV4_FRONT || (A.x.mode == KV4_SHARED && q.from < 0)) {
        const int tag = *(volatile int *) &A.x.sync[0] + 1;        // of this call; what earlier ones left has others
        if (A.x.mode == KV4_SHARED) {
            if (writes) A.x.ml[at] = make_float4(m, l, __int_as_float(tag), __int_as_float(~tag));
            r.own = 1.f;
            r.put = A.x.o + at * D;
            return r;
        }
        const float4 p = A.x.ml[at];
        if (__float_as_int(p.z) != tag || __float_as_int(p.w) != ~tag) {           // a query beyond the first max_q of its sequence
            r.skip = true;
            return r;
        }
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
// KV4_FRONT: a CTA of the call's last kernel has ended (one thread says so, and its others behind a barrier): behind the last of them the call has
__device__ __forceinline__ void kv4_leave(const Kv4Attn & A) {
    if (A.x.mode != KV4_FRONT) return;
    __threadfence();
    if (atomicAdd(&A.x.sync[1], 1) == (int) gridDim.x - 1) {
        A.x.sync[1] = 0;
        A.x.sync[0] = A.x.sync[0] + 1;
    }
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
