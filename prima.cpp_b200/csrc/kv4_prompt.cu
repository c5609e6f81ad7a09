// prima.cpp_b200/csrc/kv4_prompt.cu — attention over the 4-bit cache (kv4.cuh) for sequences with many query rows, on the 5th-generation tensor cores.
//
// Mathematics.  S = Q K^T, P = 2^(S c - reference), O += P V, divided by the row's sum at the end.  Keys and values are f16 numbers exactly; queries become f16 (a row by a power of two:
// 16-bit ones exactly, F32 as two numbers, 22 bits), weights f16 (F32: two numbers).  A row's reference is the largest score of its first tile; it moves only where a
// score lies beyond it (16 bits: by more than 2^6), and then its sum and O are scaled.
//
// Work.  An item is a (sequence, kv head, tile of query rows: tokens x heads of the group).  Two softmax groups keep the tensor cores busy in turns: with 16 bits each has 128 rows, which
// share each expanded key tile; with F32 both have the same 128 rows and every other key tile, and their sums are joined at the end.  Key tiles are two pages.  CTAs (one to an SM) take
// items by tickets, long ones of a sequence first; where there are fewer items than SMs, long items are cut into pieces, which a second kernel adds up in their order.
//   warps 0 - 3    expand: a thread has a cell's row of keys, then one of values: raw words in registers a tile ahead, f16 into the swizzle-128B images, two stages each
//   warps 4 - 11   softmax, groups of four: a thread has a row of S, which is also a lane of tensor memory
//   warp 12        MMA issuer, owner of the tensor memory, and of the tickets
// Tensor memory: S / P of either group at 0 and 256, O at 128 and 384.  Weights lie over their scores: 16 columns for 32, F32's low parts in the other 16.
// F32: every 256 cells of a group O is added to a sum in the workspace, and begins anew with a reference of its own.
//
// Bound: with 16 bits a key tile takes 4400 clocks for 256 rows: MMAs 2100 (S with both operands in shared memory, which also takes the expanded tiles), exponentials 2050 a scheduler, two
// softmax groups and expansion side by side, each group waiting for a third of it on its own two products; an item adds 12000 for queries, first tile, output; a launch 4000, or 8000 where
// items are cut.  us: 2048 tokens of 32 heads over 8 56 (610 TFLOP/s of visible pairs; over an f16 cache k_attn_prefill_tc takes 58), a plain form of elementary operations 3066; 512 behind
// 8000 cells 109 (F32 178); F32, 1077 queries behind up to 5077 cells 82 (with the sequence of one query and the join; 69 with sums that stay in tensor memory), 5200.
// On the way, us at 2048 tokens: scores 32 at a time, waited for, masks within the passes 124; the next 32 on their way 102; masks in a pass of their own over edge tiles (their code was a
// third of what was fetched and not run) 64; eight numbers of a query to a lane 57.  A row to a thread for the queries is no faster (its loads are 256 bytes apart),
// weights handed over in halves neither (F32, with sums that stay, 70 -> 77: the issuing warp waits for one group's while the other's are there).
// Error against 64 bits with F32: 3.5e-7 at 128 cells, 1.1e-6 at 4000 and more (KP_CHUNK).  With 16 bits O is the sum of all tiles, of which MMAs cut off what they add to: 2e-4 at 131 000 cells.
// A chunk's sum goes through L2, 128 KB read and written by an SM for both groups; asking for it ahead of a wait changes nothing.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cfloat>
#include <climits>
#include <type_traits>

#include "../../include/prima_b200.h"
#include "kv4_attn.cuh"

namespace pb {
namespace {

constexpr int KP_THREADS = 13 * 32, KP_TILE = 128, KP_BLOCK = 16384;   // a block: 128 rows of 64 entries
constexpr int KP_CUT_SEQ = 32, KP_CUT_TILES = KV4_MAX_CTAS + KP_CUT_SEQ;     // where long items may be cut: sequences, row tiles
// A row's reference may fall behind its largest score by 2^SLACK; a weight is 2^(15 - SLACK) at its reference, so 2^15 at most, and what f16 (F32: its low part) rounds off is 2^(SLACK - 40) of the
// row's largest weight (F32, whose references are whole numbers: 2^-39).  8, as it was with 2^6 in front of weights, lost small ones beside a large one (of weights 2^-24 of it, 2e-3); us, 512
// tokens behind 8000 in f16, 8 / 6 / 5 / 4: 110 / 110 / 111 / 112; the ragged case in F32, with four tiles to a chunk (below), 4 / 2 / 0: 75 / 77 / 77.
template <typename T> constexpr float kp_slack() { return std::is_same<T, float>::value ? 0.f : 6.f; }
// F32: key tiles of a group (256 cells) whose products add up in tensor memory, before they go to a sum in 32 bits: the tensor core cuts off what it adds to.  Error, 8 x 512 queries of 4096 cells
// (elementary 32-bit operations 1.3e-6), and us: 1 0.8e-6, 400; 2 1.1e-6, 335; 3 1.3e-6, 318; 4 1.6e-6, 308; all of them 4.9e-6, 272.  779 queries of up to 1260 cells (0.7e-6): 2 0.9e-6, 4 1.3e-6.
constexpr int KP_CHUNK = 2;
template <typename T> constexpr int kp_rows() { return std::is_same<T, float>::value ? KP_TILE : 2 * KP_TILE; }   // of an item

struct KpPiece {               // what a ticket stands for
    int s, hk, row0, rows;     // sequence, kv head, first row (of the sequence's) and rows of the tile
    int a, b, tiles;           // key tiles [a, b) of the item's
    int slot, part, parts;     // of its part in the workspace (-1: the whole item), which of how many
    Kv4Seq q;                  // pages that the tile's rows see
    int p_lo, p_hi;            // positions of the tile's first and last row
};
// of a launch whose long items may be cut, in shared memory (in registers it takes them from all roles): a sequence's rows; which one is i-th in the order of lengths, and how many row tiles
// that and those in front have; the row tiles' key tiles; how long pieces may be, 0 where items stay whole
struct KpPlan {
    int64_t q0[KP_CUT_SEQ];
    int n_q[KP_CUT_SEQ], p0[KP_CUT_SEQ], n_rows[KP_CUT_SEQ], from[KP_CUT_SEQ], ends[KP_CUT_SEQ], lens[KP_CUT_TILES], limit;
    int2 front[KP_CUT_SEQ];                                    // with X: `keep` and `from`
    template <bool X> __device__ __forceinline__ Kv4Seq seq(int s) const {       // without its pages
        Kv4Seq q{};
        q.q0 = q0[s]; q.n_q = n_q[s]; q.p0 = p0[s]; q.n_rows = n_rows[s];
        if (X) { q.keep = front[s].x; q.from = front[s].y; }
        return q;
    }
};
template <int D> struct KpPart { float o[2 * KP_TILE][D]; float m[2 * KP_TILE], l[2 * KP_TILE]; };
template <int D> struct KpSmem {
    uint8_t q[2][D / 64][KP_BLOCK];            // 16 bits: either row tile; F32: high and low
    uint8_t k[2][D / 64][KP_BLOCK], v[2][D / 64][KP_BLOCK];
    uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_full[2];
    KpPiece piece[2];          // the one at hand and the next
    float mult[2 * KP_TILE], other[2][KP_TILE];
    int cell[4][2];            // first cells of a key tile's pages (of none: -1)
    uint32_t tmem_base;
    int abort, more[2];
    KpPlan plan;
};
// tickets: words that are zero between calls.  cut: long items may be
struct KpWork { int most_rows; int * tickets; void * parts; int * abort_flag; int cut; };
enum { KP_DRAWN, KP_DONE, KP_CUT, KP_JOINED };             // tickets drawn, CTAs that are through; items that were cut, joining CTAs that are through
template <int D> struct KpParts { KpPart<D> part[KV4_SLOTS]; KpPiece item[KV4_SLOTS]; };   // item: those that were cut, their first pieces

// the tile's rows [row0, row0 + rows) of a sequence: positions and pages
template <bool X>
__device__ __forceinline__ void kp_span(const Kv4Attn & A, const Kv4Seq & q, int s, KpPiece & p) {
    p.p_lo = kv4_pos<X>(A, q, p.row0 / A.group);
    p.p_hi = kv4_pos<X>(A, q, (p.row0 + p.rows - 1) / A.group);
    p.q = q;
    kv4_span<X>(A, p.p_lo, p.p_hi, p.q);
    if (X && A.x.mode == KV4_FRONT && A.x.few > 0 && kv4_walks(A, s, q.q0 + p.row0 / A.group, q.q0 + (p.row0 + p.rows - 1) / A.group)) p.q.pages = 1;     // rows that are not written
    p.tiles = (p.q.pages + 1) / 2;
}
// Items, their pieces and slots, in the order of tickets: sequences, tiles from the last on, heads, pieces; every CTA counts them in the same way.  Where long items may be cut there are
// 32 sequences at most, of which those with the longest items come first.
__device__ __forceinline__ int kp_pieces(int tiles, int limit) { return 4 * (int64_t) tiles > 5 * (int64_t) limit ? 1 + (int) (((float) tiles - 0.5f) * __frcp_rn((float) limit)) : 1; }
__device__ __forceinline__ int warp_running_sum(int x) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, x, o);
        if ((int) (threadIdx.x & 31) >= o) x += u;
    }
    return x;
}
template <int ROWS, bool X>
__device__ __forceinline__ void kp_plan(const Kv4Attn & A, const KpWork & W, int ctas, KpPlan & plan) {     // by a warp
    const int lane = threadIdx.x & 31;
    if (lane == 0) plan.limit = 0;
    if (!W.cut) return;
    const Kv4Seq own = kv4_seq<X>(A, lane, W.most_rows, true);
    plan.q0[lane] = own.q0; plan.n_q[lane] = own.n_q; plan.p0[lane] = own.p0; plan.n_rows[lane] = own.n_rows;
    if (X) plan.front[lane] = make_int2(own.keep, own.from);
    const int len = own.n_q > 0 ? own.p0 + own.n_q : INT_MIN;
    int rank = lane < A.n_seq ? 0 : lane;
    for (int i = 0; i < A.n_seq; i++) {
        const int other = __shfl_sync(0xffffffffu, len, i);
        if (lane < A.n_seq) rank += other > len || (other == len && i < lane);
    }
    plan.from[rank] = lane;
    __syncwarp();
    const int from = plan.from[lane], ends = warp_running_sum(__shfl_sync(0xffffffffu, own.n_q > 0 ? (own.n_rows + ROWS - 1) / ROWS : 0, from));
    plan.ends[lane] = ends;
    const int all = __shfl_sync(0xffffffffu, ends, 31);
    if (all > KP_CUT_TILES) return;                   // (starts that are in no order)
    int sum = 0;
    for (int m0 = 0; m0 < all; m0 += 32) {
        const int m = m0 + lane;
        int r = 0;                                    // how many sequences end in front of tile m
#pragma unroll
        for (int step = 16; step > 0; step >>= 1)
            if (__shfl_sync(0xffffffffu, ends, r + step - 1) <= m) r += step;
        r = min(r, 31);
        KpPiece p{};
        p.row0 = (__shfl_sync(0xffffffffu, ends, r) - 1 - m) * ROWS;
        const int src = __shfl_sync(0xffffffffu, from, r);
        if (m < all) {
            const Kv4Seq q = plan.seq<X>(src);
            p.rows = min(ROWS, q.n_rows - p.row0);
            kp_span<X>(A, q, src, p);
            plan.lens[m] = p.tiles;
            sum += p.tiles;
        }
    }
    sum = __reduce_add_sync(0xffffffffu, sum) * A.cache.n_head_kv;
    __syncwarp();
    // of the even share, 4 / 3 and 2 of it that which ends first
    const int share = max(4, (sum + ctas - 1) / ctas);
    int best = share, best_cost = INT_MAX;
#pragma unroll 1
    for (int i = 0; i < 3; i++) {
        const int limit = share + (i == 0 ? 0 : i == 1 ? (share + 2) / 3 : share);
        int n = 0, most = 0;
        for (int m = lane; m < all; m += 32) {
            const int k = kp_pieces(plan.lens[m], limit);
            n += k;
            most = max(most, (int) (((float) plan.lens[m] - 0.5f) * __frcp_rn((float) k)) + 1);
        }
        n = __reduce_add_sync(0xffffffffu, n) * A.cache.n_head_kv;
        most = __reduce_max_sync(0xffffffffu, most);
        // a piece's start and end are about three tiles; rounds of the longest, or, where lengths differ, long ones first: 4 / 3 of the mean at most
        const int mean = (int) (((float) sum + 3.f * (float) n) * (4.f / 3.f) * __frcp_rn((float) ctas)) + 1, cost = min((n + ctas - 1) / ctas * (most + 3), max(most + 3, mean));
        if (cost < best_cost) { best = limit; best_cost = cost; }
    }
    if (lane == 0) plan.limit = best;
}
// by a warp: what ticket t stands for; false: there is none
template <int ROWS, bool X>
__device__ __forceinline__ bool kp_find(const Kv4Attn & A, const KpWork & W, const KpPlan & plan, int t, KpPiece & out) {
    const int lane = threadIdx.x & 31, hks = A.cache.n_head_kv;
    int before = 0, cut = 0;
    if (W.cut && plan.limit > 0) {
        const int limit = plan.limit, all = plan.ends[31];
        for (int m0 = 0; m0 < all; m0 += 32) {
            const int tiles = m0 + lane < all ? plan.lens[m0 + lane] : 0, k = tiles > 0 ? kp_pieces(tiles, limit) : 0, c = k > 1 ? k * hks : 0;
            const int x = warp_running_sum(k * hks), y = warp_running_sum(c);
            const uint32_t in = __ballot_sync(0xffffffffu, t < before + x);
            if (!in) {
                before += __shfl_sync(0xffffffffu, x, 31);
                cut += __shfl_sync(0xffffffffu, y, 31);
                continue;
            }
            const int at = __ffs((int) in) - 1, m = m0 + at, r = __popc(__ballot_sync(0xffffffffu, plan.ends[lane] <= m));
            if (lane == at) {
                KpPiece p{};
                p.row0 = (plan.ends[r] - 1 - m) * ROWS;
                p.s = plan.from[r];
                const Kv4Seq q = plan.seq<X>(p.s);
                p.rows = min(ROWS, q.n_rows - p.row0);
                kp_span<X>(A, q, p.s, p);
                const int i = t - before - (x - k * hks);
                p.hk = i / k;
                p.part = i - p.hk * k;
                p.parts = k;
                p.a = (int) ((long long) p.tiles * p.part / k);
                p.b = (int) ((long long) p.tiles * (p.part + 1) / k);
                p.slot = k > 1 ? cut + (y - c) + i : -1;
                out = p;
            }
            __syncwarp();
            return true;
        }
        return false;
    }
    for (int s0 = 0; s0 < A.n_seq; s0 += 32) {
        const Kv4Seq q = kv4_seq<X>(A, s0 + lane, W.most_rows, true);
        const int n = q.n_q > 0 ? (q.n_rows + ROWS - 1) / ROWS * hks : 0;
        const int x = warp_running_sum(n);
        const uint32_t in = __ballot_sync(0xffffffffu, t < before + x);
        if (!in) {
            before += __shfl_sync(0xffffffffu, x, 31);
            continue;
        }
        if (lane == __ffs((int) in) - 1) {
            const int i = t - before - (x - n), tile = i / hks;
            KpPiece p{};
            p.s = s0 + lane;
            p.row0 = ((q.n_rows + ROWS - 1) / ROWS - 1 - tile) * ROWS;
            p.rows = min(ROWS, q.n_rows - p.row0);
            kp_span<X>(A, q, p.s, p);
            p.hk = i - tile * hks;
            p.b = p.tiles;
            p.parts = 1;
            p.slot = -1;
            out = p;
        }
        __syncwarp();
        return true;
    }
    return false;
}

__device__ __forceinline__ uint32_t hu(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
__device__ __forceinline__ __half2 uh(uint32_t u) { return *reinterpret_cast<__half2 *>(&u); }
// waits for loads from tensor memory; what v holds may be used behind it only
#define TMEM_ARRIVED(v) \
    asm volatile("tcgen05.wait::ld.sync.aligned;" \
                 : "+r"((v)[0]), "+r"((v)[1]), "+r"((v)[2]), "+r"((v)[3]), "+r"((v)[4]), "+r"((v)[5]), "+r"((v)[6]), "+r"((v)[7]), "+r"((v)[8]), "+r"((v)[9]), "+r"((v)[10]), "+r"((v)[11]), "+r"((v)[12]), "+r"((v)[13]), "+r"((v)[14]), "+r"((v)[15]), \
                   "+r"((v)[16]), "+r"((v)[17]), "+r"((v)[18]), "+r"((v)[19]), "+r"((v)[20]), "+r"((v)[21]), "+r"((v)[22]), "+r"((v)[23]), "+r"((v)[24]), "+r"((v)[25]), "+r"((v)[26]), "+r"((v)[27]), "+r"((v)[28]), "+r"((v)[29]), "+r"((v)[30]), "+r"((v)[31]) \
                 : \
                 : "memory")
// eight numbers (four to a half-word, the halves' i-th next to each other) times their scale, as f16
__device__ __forceinline__ uint4 expand(uint32_t w, __half2 d) {
    const uint32_t s = w >> 8;
    const __half2 e = __float2half2_rn(1032.f), o = __float2half2_rn(72.f);
    return make_uint4(hu(__hmul2(__hsub2(uh((w & 0x000f000fu) | 0x64006400u), e), d)), hu(__hmul2(__hsub2(uh((w & 0x00f000f0u) | 0x54005400u), o), d)),
                      hu(__hmul2(__hsub2(uh((s & 0x000f000fu) | 0x64006400u), e), d)), hu(__hmul2(__hsub2(uh((s & 0x00f000f0u) | 0x54005400u), o), d)));
}
template <typename T, int D, bool X>
__global__ void __launch_bounds__(KP_THREADS, 1) k_kv4_attn_prompt(const __grid_constant__ Kv4Attn A, const __grid_constant__ KpWork W) {
    constexpr bool F32 = std::is_same<T, float>::value;
    constexpr int ROWS = kp_rows<T>(), NB = D / 32;
    constexpr float SLACK = kp_slack<T>(), UP = 15.f - SLACK;
    extern __shared__ uint8_t smem_raw[];
    KpSmem<D> & S = *reinterpret_cast<KpSmem<D> *>(smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    volatile int * cta_abort = &S.abort;
    if (warp == 12) {
        if (lane == 0) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                mbar_init(&S.k_full[i], 4);
                mbar_init(&S.v_full[i], 4);
                mbar_init(&S.k_empty[i], 1);
                mbar_init(&S.v_empty[i], 1);
                mbar_init(&S.s_full[i], 1);
                mbar_init(&S.p_full[i], 4);
                mbar_init(&S.o_full[i], 1);
            }
            S.abort = 0;
            mbar_fence_init();
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        __syncwarp();
        tmem_alloc(&S.tmem_base, 512);
    }
    int ticket = blockIdx.x;
    if (warp == 12) {
        kp_plan<ROWS, X>(A, W, gridDim.x, S.plan);
        __syncwarp();
        const bool more = kp_find<ROWS, X>(A, W, S.plan, ticket, S.piece[0]);
        if (lane == 0) S.more[0] = more;
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *(volatile uint32_t *) &S.tmem_base;
    if (X) pdl_trigger();                          // the join's CTAs may come where this kernel has none at work any more
    uint32_t tiles = 0, pieces = 0, of_group[2] = {0, 0}, ends[2] = {0, 0};   // key tiles and pieces in front; key tiles and ends of chunks of either group (all roles count them)
    while (*(volatile int *) &S.more[pieces & 1]) {
        const KpPiece & P = S.piece[pieces & 1];
        const int2 hole = kv4_hole<X>(A, P.q);
        const int n = P.b - P.a, groups = (F32 ? n > 1 : P.rows > KP_TILE) ? 2 : 1;      // groups at work
        if (warp < 4) {
            // ---- expand ----
            const int x = threadIdx.x, half = x >> 6, t6 = x & 63, r = t6, tv = (r & ~7) | ((r & 3) << 1) | ((r >> 2) & 1);
            constexpr int WORDS = NB == 4 ? 4 : 2;                 // of a quarter of a row
            uint32_t kw[4][WORDS], vw[4][WORDS], ks[NB], vs[NB];
            auto chunk_of = [&](int j) {                          // this half's page of tile j, none: null
                const int i = 2 * (P.a + j) + half;
                const int id = j < n && i < P.q.pages ? kv4_page<X>(A, P.q, P.s, i) : -1;
                return id >= 0 ? kv4_chunk<D>(A.cache, id, P.hk) : nullptr;
            };
            auto rows_of = [&](const uint8_t * row, const uint8_t * scales, uint32_t (&w)[4][WORDS], uint32_t (&d)[NB]) {
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    if constexpr (NB == 4) *reinterpret_cast<uint4 *>(w[c]) = row ? *reinterpret_cast<const uint4 *>(row + 16 * c) : make_uint4(0u, 0u, 0u, 0u);
                    else *reinterpret_cast<uint2 *>(w[c]) = row ? *reinterpret_cast<const uint2 *>(row + 8 * c) : make_uint2(0u, 0u);
                }
                if constexpr (NB == 4) *reinterpret_cast<uint4 *>(d) = row ? *reinterpret_cast<const uint4 *>(scales) : make_uint4(0u, 0u, 0u, 0u);
                else *reinterpret_cast<uint2 *>(d) = row ? *reinterpret_cast<const uint2 *>(scales) : make_uint2(0u, 0u);
            };
            const uint8_t * now = chunk_of(0), * later = chunk_of(1);
            auto ask_k = [&](const uint8_t * p) { rows_of(p ? p + t6 * (D / 2) : nullptr, p + 2 * kv4_rows_bytes(D) + kv4_scale(D, t6 & ~1, 0), kw, ks); };
            auto ask_v = [&](const uint8_t * p) {
                rows_of(p ? p + kv4_rows_bytes(D) + r * (D / 2) : nullptr, p + 2 * kv4_rows_bytes(D) + kv4_scales_bytes(D) + kv4_scale(D, tv & ~1, 0), vw, vs);
            };
            ask_k(now);
            ask_v(now);
            for (int j = 0; j < n; j++) {
                const uint32_t u = tiles + (uint32_t) j;
                const int st = (int) (u & 1);
                const uint8_t * third = chunk_of(j + 2);
                if (t6 == 0) S.cell[u & 3][half] = now ? kv4_page_index<X>(A, P.q, 2 * (P.a + j) + half) * KV4_CELLS : -1;
                if (u >= 2) mbar_wait(&S.k_empty[st], (u / 2 - 1) & 1, cta_abort, W.abort_flag);
                {
                    const uint32_t odd = t6 & 1 ? 0x3232u : 0x1010u;
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        const __half2 d = uh(__byte_perm(ks[b], 0u, odd));
#pragma unroll
                        for (int c = 0; c < 4; c++) *reinterpret_cast<uint4 *>(S.k[st][b >> 1] + x * 128 + ((((b & 1) * 4 + c) ^ (x & 7)) << 4)) = expand(kw[c][b], d);
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&S.k_full[st]);
                ask_k(later);
                if (u >= 2) mbar_wait(&S.v_empty[st], (u / 2 - 1) & 1, cta_abort, W.abort_flag);
                {
                    const int i = 2 * (P.a + j) + half, cell = kv4_page_index<X>(A, P.q, i) * KV4_CELLS + tv, t = half * 64 + tv;
                    // a weight of zero does not silence a scale that is no number: cells nobody sees may hold anything
                    const bool seen = cell <= P.p_hi && (A.window <= 0 || P.p_lo - cell < A.window || cell < A.first) && !kv4_in_hole<X>(hole, cell);
                    const uint32_t odd = tv & 1 ? 0x3232u : 0x1010u;
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        const __half2 d = uh(seen ? __byte_perm(vs[b], 0u, odd) : 0u);
#pragma unroll
                        for (int c = 0; c < 4; c++) {
                            // words 2c, 2c+1 of the row: half-word b of either
                            const uint32_t w = __byte_perm(vw[c][b / 2], vw[c][WORDS / 2 + b / 2], b & 1 ? 0x7632 : 0x5410);
                            const int q = c ^ (2 * ((r >> 1) & 1));
                            *reinterpret_cast<uint4 *>(S.v[st][b >> 1] + t * 128 + ((((b & 1) * 4 + q) ^ (t & 7)) << 4)) = expand(w, d);
                        }
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&S.v_full[st]);
                ask_v(later);
                now = later;
                later = third;
            }
        } else if (warp == 12) {
            // ---- MMA ----
            constexpr uint32_t idesc = (1u << 4) | ((uint32_t) (128 >> 3) << 17) | ((uint32_t) (128 >> 4) << 24);
            constexpr uint32_t idesc_v = (1u << 4) | ((uint32_t) (D >> 3) << 17) | ((uint32_t) (128 >> 4) << 24) | (1u << 16);
            asm volatile("bar.sync 4, 288;" ::: "memory");        // the queries are there
            // S of a tile behind the P V that reads this tensor memory (MMAs run in order)
            auto scores = [&](int grp, uint32_t u) {
                const int st = (int) (u & 1);
                if (F32 || grp == 0) mbar_wait(&S.k_full[st], (u / 2) & 1, cta_abort, W.abort_flag);
                __syncwarp();
                fence_after();
                if (elect_one()) {
#pragma unroll
                    for (int part = 0; part < (F32 ? 2 : 1); part++) {   // F32: the low parts first: every product is aligned to the sum so far and cut off (1.4e-6 -> 1.1e-6)
                        const uint64_t dq = desc_sw128(smem_u32(S.q[F32 ? 1 - part : grp])), dk = desc_sw128(smem_u32(S.k[st]));
#pragma unroll
                        for (int k = 0; k < D / 16; k++)
                            mma_f16<1>(tmem + 256 * grp, dq + (k >> 2) * (KP_BLOCK >> 4) + 2 * (k & 3), dk + (k >> 2) * (KP_BLOCK >> 4) + 2 * (k & 3), idesc, (uint32_t) ((part | k) != 0));
                    }
                    mma_commit(&S.s_full[grp]);
                    if (F32 || grp == groups - 1) mma_commit(&S.k_empty[st]);
                }
                __syncwarp();
            };
            auto values = [&](int grp, uint32_t u, int i, bool last) {       // i: which of the group's tiles
                const int st = (int) (u & 1);
                if (F32 || grp == 0) mbar_wait(&S.v_full[st], (u / 2) & 1, cta_abort, W.abort_flag);
                mbar_wait(&S.p_full[grp], (of_group[grp] + (uint32_t) i) & 1, cta_abort, W.abort_flag);
                __syncwarp();
                fence_after();
                if (elect_one()) {
                    const uint64_t dv = desc_sw128_mn(smem_u32(S.v[st]), KP_BLOCK);
#pragma unroll
                    for (int part = 0; part < (F32 ? 2 : 1); part++)
#pragma unroll
                        for (int k = 0; k < 8; k++)
                            mma_f16_ts(tmem + 256 * grp + 128, tmem + 256 * grp + 32 * (k >> 1) + 8 * (k & 1) + 16 * part, dv + k * (2048 >> 4), idesc_v, (uint32_t) (((F32 ? i % KP_CHUNK : i) | part | k) != 0));
                    if (last || (F32 && i % KP_CHUNK == KP_CHUNK - 1)) mma_commit(&S.o_full[grp]);
                    if (F32 || grp == groups - 1) mma_commit(&S.v_empty[st]);
                }
                __syncwarp();
            };
            if constexpr (F32) {
                for (int j = -2; j < n; j++) {
                    if (j >= 0) values(j & 1, tiles + (uint32_t) j, j >> 1, j + 2 >= n);
                    if (j + 2 < n) scores(j & 1, tiles + (uint32_t) (j + 2));
                }
            } else {
                for (int j = -1; j < n; j++)
                    for (int grp = 0; grp < groups; grp++) {
                        if (j >= 0) values(grp, tiles + (uint32_t) j, j, j == n - 1);
                        if (j + 1 < n) scores(grp, tiles + (uint32_t) (j + 1));
                    }
            }
            if (lane == 0) ticket = (int) gridDim.x + atomicAdd(&W.tickets[KP_DRAWN], 1);
            ticket = __shfl_sync(0xffffffffu, ticket, 0);
            const int later = (pieces + 1) & 1;
            const bool more = kp_find<ROWS, X>(A, W, S.plan, ticket, S.piece[later]);         // beside the piece's end; earlier, and CTAs with long pieces would draw more
            if (lane == 0) S.more[later] = more;
        } else {
            // ---- softmax ----
            const int grp = (warp - 4) >> 2, quad = warp & 3, row = quad * 32 + lane;       // (the quarter of tensor memory that a warp reaches is its number's last two bits)
            const int rows0 = F32 ? 0 : grp * KP_TILE;                                        // the group's first row of the item
            // this lane's row: its token and head, and where they lie (others' by shuffles: a division costs more than a row)
            const int at = P.row0 + rows0 + row, tok = at / A.group, head = P.hk * A.group + at - tok * A.group;
            const bool mine_is = rows0 + row < P.rows;
            const uint32_t valid = __ballot_sync(0xffffffffu, mine_is);
            const int64_t q_at = (P.q.q0 + tok) * A.ldq + (int64_t) head * D;
            // queries -> f16 in the swizzle-128B image: 8 numbers to a lane; a row's largest comes to 2^13 .. 2^14.  F32: half of a warp's rows are its sister's
            {
                constexpr int LPR = D / 8, RPW = 32 / LPR, PASSES = 32 / RPW / (F32 ? 2 : 1), ONCE = PASSES < 8 ? PASSES : 8;    // lanes to a row, rows at once
                const int sub = lane / LPR, l8 = lane % LPR;
#pragma unroll 1
                for (int i0 = 0; i0 < PASSES; i0 += ONCE) {
                    float4 v[ONCE][2];
#pragma unroll
                    for (int i = 0; i < ONCE; i++) {
                        const int rr = (i0 + i + (F32 ? grp * PASSES : 0)) * RPW + sub;
                        const T * from = (const T *) A.q + __shfl_sync(0xffffffffu, q_at, rr) + 8 * l8;
                        v[i][0] = valid >> rr & 1 ? load4(from) : make_float4(0.f, 0.f, 0.f, 0.f);
                        v[i][1] = valid >> rr & 1 ? load4(from + 4) : make_float4(0.f, 0.f, 0.f, 0.f);
                    }
#pragma unroll
                    for (int i = 0; i < ONCE; i++) {
                        const int rr = quad * 32 + (i0 + i + (F32 ? grp * PASSES : 0)) * RPW + sub;
                        float4 x = v[i][0], y = v[i][1];
                        float top = fmaxf(fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))), fmaxf(fmaxf(fabsf(y.x), fabsf(y.y)), fmaxf(fabsf(y.z), fabsf(y.w))));
#pragma unroll
                        for (int o = LPR / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                        const int ex = top > 0.f && top < INFINITY ? min(126, 140 - (int) (__float_as_uint(top) >> 23)) : 0;
                        const float up = __int_as_float((ex + 127) << 23) * (A.scale < 0.f ? -1.f : 1.f);
                        // scores in units of log2; never 0: a masked score stays -inf
                        if (l8 == 0) S.mult[rows0 + rr] = fmaxf(fabsf(A.scale) * 1.4426950408889634f * __int_as_float((127 - ex) << 23), FLT_MIN);
                        x.x *= up; x.y *= up; x.z *= up; x.w *= up; y.x *= up; y.y *= up; y.z *= up; y.w *= up;
                        const __half2 h[4] = {__floats2half2_rn(x.x, x.y), __floats2half2_rn(x.z, x.w), __floats2half2_rn(y.x, y.y), __floats2half2_rn(y.z, y.w)};
                        const int to = (l8 >> 3) * KP_BLOCK + rr * 128 + (((l8 & 7) ^ (rr & 7)) << 4);
                        *reinterpret_cast<uint4 *>(&S.q[F32 ? 0 : grp][0][0] + to) = make_uint4(hu(h[0]), hu(h[1]), hu(h[2]), hu(h[3]));
                        if constexpr (F32) {
                            const float2 b[4] = {__half22float2(h[0]), __half22float2(h[1]), __half22float2(h[2]), __half22float2(h[3])};
                            *reinterpret_cast<uint4 *>(&S.q[1][0][0] + to) =
                                make_uint4(hu(__floats2half2_rn(x.x - b[0].x, x.y - b[0].y)), hu(__floats2half2_rn(x.z - b[1].x, x.w - b[1].y)),
                                           hu(__floats2half2_rn(y.x - b[2].x, y.y - b[2].y)), hu(__floats2half2_rn(y.z - b[3].x, y.w - b[3].y)));
                        }
                    }
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            asm volatile("bar.sync 4, 288;" ::: "memory");
            if (grp < groups) {
                const int pos = mine_is ? kv4_pos<X>(A, P.q, tok) : -1;
                const float c = S.mult[rows0 + row];
                const uint32_t mine = tmem + ((uint32_t) (quad * 32) << 16) + 256 * grp;
                const int g_lo = kv4_pos<X>(A, P.q, (P.row0 + rows0) / A.group);              // of the group's first row
                float m = -INFINITY, l = 0.f;
                float t[2][32];                                    // scores, 32 being worked on and 32 on their way
                uint32_t * const t0 = reinterpret_cast<uint32_t *>(t[0]), * const t1 = reinterpret_cast<uint32_t *>(t[1]);
                // F32: the sum of the chunks in front, a thread's own: numbers 4 k .. 4 k + 3 of row r at 128 k + r
                float m_far = -INFINITY, l_far = 0.f, f_far = 0.f, f_own = 1.f;
                float4 * const far = reinterpret_cast<float4 *>(reinterpret_cast<KpParts<D> *>(W.parts)->part[F32 ? 2 * blockIdx.x + grp : 0].o[KP_TILE]) + row;
                auto ask_far = [&](int h) {                        // numbers h .. h + 31 of it -> t[1]
#pragma unroll
                    for (int k = 0; k < 8; k++) *reinterpret_cast<float4 *>(&t[1][4 * k]) = far[(h / 4 + k) * KP_TILE];
                };
                auto factors = [&] {                               // of the sum in front and of the chunk at hand, which become one
                    const float top = fmaxf(m_far, m);
                    f_far = part_factor(m_far, l_far, top);
                    f_own = part_factor(m, l, top);
                    l_far = l_far * f_far + l * f_own;
                    m_far = top;
                };
                for (int j = F32 ? grp : 0, i = 0; j < n; j += F32 ? 2 : 1, i++) {
                    mbar_wait(&S.s_full[grp], (of_group[grp] + (uint32_t) i) & 1, cta_abort, W.abort_flag);
                    __syncwarp();
                    fence_after();
                    // (four of them: written for tile j + 4 behind the scores of j + 2, which come behind the weights of j)
                    const int c0 = *(volatile int *) &S.cell[(tiles + (uint32_t) j) & 3][0], c1 = *(volatile int *) &S.cell[(tiles + (uint32_t) j) & 3][1];
                    const bool whole = min(c0, c1) >= 0 && max(c0, c1) <= g_lo - 63 && (A.window <= 0 || (P.p_hi - c0 < A.window || c0 + 63 < A.first) && (P.p_hi - c1 < A.window || c1 + 63 < A.first)) && !kv4_has_hole<X>(hole, c0) && !kv4_has_hole<X>(hole, c1);
                    if (!whole) {   // a score that is not seen is -inf: in its place, ahead of the passes over the tile
                        const int from = A.window > 0 ? max(0, pos - A.window + 1) : 0;
#pragma unroll 1
                        for (int h = 0; h < 4; h++) {
                            const int page = h < 2 ? c0 : c1, base = page + 32 * (h & 1);
                            auto below = [&](int cell) { const int k = cell - base; return k <= 0 ? 0u : k >= 32 ? 0xffffffffu : (1u << k) - 1u; };     // cells in front of it
                            uint32_t seen = page < 0 || base > pos ? 0u : below(pos + 1) & (~below(from) | below(A.first));
                            if (X && hole.y > 0) seen &= below(hole.x) | ~below(hole.y);
                            TMEM_LD32(mine + 32 * h, t0);
                            TMEM_ARRIVED(t0);
#pragma unroll
                            for (int i = 0; i < 32; i++) t[0][i] = seen >> i & 1 ? t[0][i] : -INFINITY;
                            TMEM_ST16(mine + 32 * h, t0);
                            TMEM_ST16(mine + 32 * h + 16, t0 + 16);
                        }
                        tmem_wait_st();
                    }
                    float tm[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                    TMEM_LD32(mine, t0);
#pragma unroll
                    for (int h = 0; h < 4; h++) {
                        if (h & 1) TMEM_ARRIVED(t1);
                        else TMEM_ARRIVED(t0);
                        if (h & 1) TMEM_LD32(mine + 32 * ((h + 1) & 3), t0);      // (behind the last: the first again)
                        else TMEM_LD32(mine + 32 * ((h + 1) & 3), t1);
                        float(&x)[32] = t[h & 1];
#pragma unroll
                        for (int i = 0; i < 32; i++) tm[i & 3] = fmaxf(tm[i & 3], x[i]);
                    }
                    // rounded upwards, so that weights stay within 2^15 however large scores are.  F32: to a whole number: what weights, sums and parts are scaled by are powers of two then
                    float top = __fmul_ru(fmaxf(fmaxf(tm[0], tm[1]), fmaxf(tm[2], tm[3])), c);
                    if (F32) top = ceilf(top);
                    const bool move = top > __fadd_rd(m, SLACK);   // (the first: m is -inf)
                    if (__any_sync(0xffffffffu, move)) {
                        const float f = !move ? 1.f : m == -INFINITY ? 0.f : ex2(m - top);
                        if (move) m = top;
                        l *= f;
                        if (F32 ? i % KP_CHUNK != 0 : i > 0) {
#pragma unroll
                            for (int h = 0; h < D; h += 32) {
                                TMEM_LD32(mine + 128 + h, t1);
                                TMEM_ARRIVED(t1);
#pragma unroll
                                for (int i = 0; i < 32; i++) t[1][i] *= f;
                                TMEM_ST16(mine + 128 + h, t1);
                                TMEM_ST16(mine + 128 + h + 16, t1 + 16);
                            }
                        }
                    }
                    const float off = m == -INFINITY ? 0.f : __fsub_rd(UP, m);
                    float e4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int h = 0; h < 4; h++) {
                        if (h & 1) TMEM_ARRIVED(t1);
                        else TMEM_ARRIVED(t0);
                        if (h < 3) {
                            if (h & 1) TMEM_LD32(mine + 32 * (h + 1), t0);
                            else TMEM_LD32(mine + 32 * (h + 1), t1);
                        }
                        float(&x)[32] = t[h & 1];
                        uint32_t p[16], lo[F32 ? 16 : 1];
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            const float a = ex2(fmaf(x[2 * i], c, off)), b = ex2(fmaf(x[2 * i + 1], c, off));
                            e4[i & 1] += a;
                            e4[2 + (i & 1)] += b;
                            const __half2 hi = __floats2half2_rn(a, b);
                            p[i] = hu(hi);
                            if constexpr (F32) {
                                const float2 back = __half22float2(hi);
                                lo[i] = hu(__floats2half2_rn(a - back.x, b - back.y));
                            }
                        }
                        TMEM_ST16(mine + 32 * h, p);               // over the scores
                        if constexpr (F32) TMEM_ST16(mine + 32 * h + 16, lo);
                    }
                    l += (e4[0] + e4[1]) + (e4[2] + e4[3]);
                    tmem_wait_st();
                    fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&S.p_full[grp]);
                    if (F32 && i % KP_CHUNK == KP_CHUNK - 1 && j + 2 < n) {       // a chunk ends: beside the next scores
                        mbar_wait(&S.o_full[grp], (ends[grp] + (uint32_t) (i / KP_CHUNK)) & 1, cta_abort, W.abort_flag);
                        __syncwarp();
                        fence_after();
                        factors();
#pragma unroll 1
                        for (int h = 0; h < D; h += 32) {
                            TMEM_LD32(mine + 128 + h, t0);
                            if (i >= KP_CHUNK) ask_far(h);
                            TMEM_ARRIVED(t0);
#pragma unroll
                            for (int k = 0; k < 32; k++) t[0][k] = i >= KP_CHUNK ? fmaf(t[1][k], f_far, t[0][k] * f_own) : t[0][k] * f_own;
#pragma unroll
                            for (int k = 0; k < 32; k += 4) far[(h + k) / 4 * KP_TILE] = make_float4(t[0][k], t[0][k + 1], t[0][k + 2], t[0][k + 3]);
                        }
                        m = -INFINITY;
                        l = 0.f;
                    }
                }
                // (all scores are made, too, before the queries' memory is used again: they come in front of the last products)
                mbar_wait(&S.o_full[grp], (ends[grp] + (uint32_t) (F32 ? ((n - grp + 1) / 2 - 1) / KP_CHUNK : 0)) & 1, cta_abort, W.abort_flag);
                __syncwarp();
                fence_after();
                constexpr int PIECE = 4, PIECES = D / PIECE;       // numbers to a piece; row r's pieces are rotated by r
                float other = 0.f;                                  // F32: factor of the other group's sum
                const bool folded = F32 && (n - grp + 1) / 2 > KP_CHUNK;
                if (folded) {
                    factors();
                    m = m_far;
                    l = l_far;
                }
                auto own_sum = [&](int h) {                         // numbers h .. h + 31 of the row's sum -> t[0]
                    TMEM_LD32(mine + 128 + h, t0);
                    if (folded) ask_far(h);
                    TMEM_ARRIVED(t0);
                    if (F32)
#pragma unroll
                        for (int k = 0; k < 32; k++) t[0][k] = folded ? fmaf(t[1][k], f_far, t[0][k] * f_own) : t[0][k] * f_own;
                };
                float * const os32 = reinterpret_cast<float *>(&S.q[0][0][0]) + row * D;
                if (F32 && groups == 2) {                           // the second group's sums go to the first through the queries' memory
                    if (grp == 1) {
#pragma unroll 1
                        for (int h = 0; h < D; h += 32) {
                            own_sum(h);
#pragma unroll
                            for (int i = 0; i < 32; i += 4) store4(os32 + ((h + i) / 4 + row) % PIECES * 4, make_float4(t[0][i], t[0][i + 1], t[0][i + 2], t[0][i + 3]));
                        }
                        S.other[0][row] = m;
                        S.other[1][row] = l;
                    }
                    asm volatile("bar.sync 5, 256;" ::: "memory");
                    if (grp == 0) {
                        const float m2 = S.other[0][row], l2 = S.other[1][row], top = fmaxf(m, m2);
                        const float f = part_factor(m, l, top);
                        other = part_factor(m2, l2, top);
                        l = l * f + l2 * other;
                        m = top;
                        f_own *= f;
                        f_far *= f;
                    }
                }
                if (!F32 || grp == 0) {
                    const float inv = P.slot >= 0 ? 1.f : l == 0.f ? 0.f : 1.f / l;
                    KpPart<D> * part = nullptr;
                    Kv4Row w{inv, 0.f, nullptr, nullptr, false};
                    if (X && A.x.mode == KV4_FRONT) pdl_wait();        // the kernel in front has the sequences' own parts
                    if (X && P.slot < 0 && mine_is) w = kv4_row<D>(A, P.q, P.q.q0 + tok, head, m - UP, l, true);
                    const uint32_t write = X ? __ballot_sync(0xffffffffu, mine_is && !w.skip) : valid;
                    if (P.slot >= 0) {
                        part = &reinterpret_cast<KpParts<D> *>(W.parts)->part[P.slot];
                        part->m[rows0 + row] = m;
                        part->l[rows0 + row] = l;
                        if (threadIdx.x == 128 && P.part == 0) reinterpret_cast<KpParts<D> *>(W.parts)->item[atomicAdd(&W.tickets[KP_CUT], 1)] = P;
                    }
                    // through the queries' memory, so that a warp stores whole rows
                    T * os = reinterpret_cast<T *>(&S.q[F32 ? 0 : grp][0][0]) + row * D;
#pragma unroll
                    for (int h = 0; h < D; h += 32) {
                        own_sum(h);
                        if (F32 && groups == 2) {
#pragma unroll
                            for (int i = 0; i < 32; i += 4) {
                                const float4 y = *reinterpret_cast<const float4 *>(os32 + ((h + i) / 4 + row) % PIECES * 4);
                                t[0][i] += y.x * other;
                                t[0][i + 1] += y.y * other;
                                t[0][i + 2] += y.z * other;
                                t[0][i + 3] += y.w * other;
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 32; i++) t[0][i] *= X ? w.own : inv;
#pragma unroll
                        for (int i = 0; i < 32; i += 8) {           // columns 0 2 4 6 | 1 3 5 7 of an eight are numbers 0 1 2 3 | 4 5 6 7
                            float4 a = make_float4(t[0][i], t[0][i + 2], t[0][i + 4], t[0][i + 6]), b = make_float4(t[0][i + 1], t[0][i + 3], t[0][i + 5], t[0][i + 7]);
                            if (part) {
                                *reinterpret_cast<float4 *>(&part->o[rows0 + row][h + i]) = a;
                                *reinterpret_cast<float4 *>(&part->o[rows0 + row][h + i + 4]) = b;
                            } else {
                                if (X && w.from) {
                                    const Kv4Row r{1.f, w.other, w.from, nullptr, false};
                                    a = kv4_mix(r, a, h + i);
                                    b = kv4_mix(r, b, h + i + 4);
                                }
                                store4(os + ((h + i) / 4 + row) % PIECES * 4, a);
                                store4(os + ((h + i) / 4 + 1 + row) % PIECES * 4, b);
                            }
                        }
                    }
                    if (!part) {
                        constexpr int LPR = D / 4, RPW = 32 / LPR;
                        const int sub = lane / LPR, l4 = lane % LPR;
                        __syncwarp();                               // a warp reads its own rows
                        const int64_t o_at = (P.q.q0 + tok) * A.ldo + (int64_t) head * D;
                        const T * rows = reinterpret_cast<const T *>(&S.q[F32 ? 0 : grp][0][0]) + quad * 32 * D;
#pragma unroll 8
                        for (int i = 0; i < 32 / RPW; i++) {
                            const int rr = i * RPW + sub;
                            const float4 v = load4(rows + rr * D + (l4 + quad * 32 + rr) % PIECES * 4);
                            const int64_t to = __shfl_sync(0xffffffffu, o_at, rr);
                            if (write >> rr & 1) store4((T *) A.out + to + 4 * l4, v);
                        }
                    }
                }
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        fence_before();
        __syncthreads();
        tiles += (uint32_t) n;
        pieces++;
        for (int grp = 0; grp < groups; grp++) {
            of_group[grp] += (uint32_t) (F32 ? (n - grp + 1) / 2 : n);
            ends[grp] += (uint32_t) (F32 ? ((n - grp + 1) / 2 - 1) / KP_CHUNK + 1 : 1);
        }
        fence_after();
    }
    pdl_wait();                                    // the end of this kernel is the end of the one in front
    if (warp == 12) {
        tmem_free(tmem, 512);
        if (lane == 0 && atomicAdd(&W.tickets[KP_DONE], 1) == (int) gridDim.x - 1) W.tickets[KP_DRAWN] = W.tickets[KP_DONE] = 0;   // the last CTA: every ticket has been drawn
        if (X && lane == 0 && !W.cut) kv4_leave(A);
    }
}

// Items that were cut, eight rows to a CTA at a time: a warp adds a row's parts in their order, a lane D / 32 numbers.
template <typename T, int D, bool X>
__global__ void __launch_bounds__(256) k_kv4_join(const __grid_constant__ Kv4Attn A, const __grid_constant__ KpWork W) {
    constexpr int PER = D / 32, ONCE = X ? 4 : 8, EIGHTS = kp_rows<T>() / 8;
    if (X) pdl_wait();
    const int lane = threadIdx.x & 31, items = *(volatile int *) &W.tickets[KP_CUT];
    const KpParts<D> & all = *reinterpret_cast<const KpParts<D> *>(W.parts);
    for (int task = blockIdx.x; task < items * EIGHTS; task += gridDim.x) {
        const KpPiece & p = all.item[task / EIGHTS];
        const int r = task % EIGHTS * 8 + (threadIdx.x >> 5), n = p.parts;
        if (r >= p.rows) continue;
        const KpPart<D> * parts = &all.part[p.slot];
        float top = -INFINITY, l = 0.f, x[PER];
        for (int i = lane; i < n; i += 32) top = fmaxf(top, parts[i].m[r]);
        top = warp_max(top);
#pragma unroll
        for (int e = 0; e < PER; e++) x[e] = 0.f;
        for (int i0 = 0; i0 < n; i0 += 32) {
            float f = 0.f, fl = 0.f;
            if (i0 + lane < n) {
                const float mi = parts[i0 + lane].m[r], li = parts[i0 + lane].l[r];
                f = part_factor(mi, li, top);
                fl = li * f;
            }
            l += warp_sum(fl);
            for (int i1 = 0; i1 < min(32, n - i0); i1 += ONCE) {
                float y[ONCE][PER];
#pragma unroll
                for (int k = 0; k < ONCE; k++) {
                    const float * o = &parts[min(i0 + i1 + k, n - 1)].o[r][lane * PER];
                    if constexpr (PER == 4) *reinterpret_cast<float4 *>(y[k]) = *reinterpret_cast<const float4 *>(o);
                    else *reinterpret_cast<float2 *>(y[k]) = *reinterpret_cast<const float2 *>(o);
                }
#pragma unroll
                for (int k = 0; k < ONCE; k++) {
                    const float h = __shfl_sync(0xffffffffu, f, i1 + k);          // (behind the last: 0)
                    if (i0 + i1 + k < n)
#pragma unroll
                        for (int e = 0; e < PER; e++) x[e] = fmaf(y[k][e], h, x[e]);
                }
            }
        }
        const float inv = X ? 1.f : l == 0.f ? 0.f : 1.f / l;
        const int at = p.row0 + r, tt = at / A.group;
        T * out = (T *) A.out + (p.q.q0 + tt) * A.ldo + (int64_t) (p.hk * A.group + at - tt * A.group) * D + lane * PER;
        if constexpr (X) {
            const Kv4Row w = kv4_row<D>(A, p.q, p.q.q0 + tt, p.hk * A.group + at - tt * A.group, top - (15.f - kp_slack<T>()), l, lane == 0);
            if (w.skip) continue;
#pragma unroll
            for (int e = 0; e < PER; e++) x[e] = w.from ? fmaf(w.from[lane * PER + e], w.other, x[e] * w.own) : x[e] * w.own;
        }
        if constexpr (PER == 4) store4(out, make_float4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv));
        else
#pragma unroll
            for (int e = 0; e < PER; e++) {
                if constexpr (std::is_same<T, float>::value) out[e] = x[e] * inv;
                else if constexpr (std::is_same<T, __half>::value) out[e] = __float2half_rn(x[e] * inv);
                else out[e] = __float2bfloat16_rn(x[e] * inv);
            }
    }
    __syncthreads();
    if (threadIdx.x == 0 && atomicAdd(&W.tickets[KP_JOINED], 1) == (int) gridDim.x - 1) W.tickets[KP_CUT] = W.tickets[KP_JOINED] = 0;
    if (X && threadIdx.x == 0) kv4_leave(A);
}

template <typename T, int D, bool X>
int prompt_launch(const Kv4Attn & a, KpWork w, cudaStream_t st, int & launches) {
    constexpr size_t smem = sizeof(KpSmem<D>) + 1024;
    static_assert(smem <= 232448, "shared memory of an SM");
    static FuncAttrCache cache;
    cudaError_t e = ensure_dyn_smem(cache, (const void *) k_kv4_attn_prompt<T, D, X>, smem, true);
    if (e != cudaSuccess) return (int) e;
    const int ctas = sm_count() < KV4_MAX_CTAS ? sm_count() : KV4_MAX_CTAS;
    // (a plan adds up key tiles of all items: in 30 bits.  An item's pages are those that the tables it walks have room for)
    const auto room = [](int64_t ld) { return ld < INT_MAX / KV4_CELLS ? ld : (int64_t) INT_MAX / KV4_CELLS; };
    const bool rest = a.x.mode == KV4_FRONT && a.x.few > 0;       // most of its rows may be those of sequences that walk, which are no work
    const int64_t items = rest ? 0 : (a.n_tokens * a.group + kp_rows<T>() - 1) / kp_rows<T>() * a.cache.n_head_kv;
    const int64_t pages = (a.x.mode != KV4_FRONT ? room(a.table_ld) : 0) + (a.x.mode != KV4_PLAIN ? room(a.x.prefix_ld) : 0);
    w.cut = a.n_seq <= KP_CUT_SEQ && items < ctas && KP_CUT_TILES * (pages / 2 + 1) * a.cache.n_head_kv < 1 << 30;
    launches += w.cut ? 2 : 1;
    // Behind the kernel of few rows (most_rows > 0), CTAs start where that has none at work: it has nothing that they read, and all in front of it has ended when it starts.  Behind another of this kernel, or
    // its join, they do not: tickets and parts are the same
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ctas); cfg.blockDim = dim3(KP_THREADS); cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = w.most_rows > 0 || (a.x.mode == KV4_FRONT && !rest) ? 1 : 0;
    e = cudaLaunchKernelEx(&cfg, k_kv4_attn_prompt<T, D, X>, a, w);
    if (e != cudaSuccess || !w.cut) return (int) e;
    cudaLaunchConfig_t join{};
    join.gridDim = dim3(4 * sm_count()); join.blockDim = dim3(256); join.stream = st;
    join.attrs = attr;
    join.numAttrs = X ? 1 : 0;
    return (int) cudaLaunchKernelEx(&join, k_kv4_join<T, D, X>, a, w);
}

}  // namespace

size_t kv4_prompt_workspace(int D) { return D == 128 ? sizeof(KpParts<128>) : sizeof(KpParts<64>); }

template <int D, bool X>
static int prompt_launch(const Kv4Attn & a, const KpWork & w, int type, cudaStream_t st, int & launches) {
    return type == PB200_TYPE_F32   ? prompt_launch<float, D, X>(a, w, st, launches)
           : type == PB200_TYPE_F16 ? prompt_launch<__half, D, X>(a, w, st, launches)
                                    : prompt_launch<__nv_bfloat16, D, X>(a, w, st, launches);
}
int launch_kv4_attn_prompt(const Kv4Attn & a, int D, int type, int most_rows, int * tickets, void * parts, cudaStream_t st, bool ext, int & launches) {
    const KpWork w{most_rows, tickets, parts, abort_flag(), 0};
    if (ext) return D == 128 ? prompt_launch<128, true>(a, w, type, st, launches) : prompt_launch<64, true>(a, w, type, st, launches);
    return D == 128 ? prompt_launch<128, false>(a, w, type, st, launches) : prompt_launch<64, false>(a, w, type, st, launches);
}

}  // namespace pb
