// prima.cpp_b200/csrc/kv4_rows.cu — attention over the 4-bit cache (kv4.cuh) for sequences with few query rows: single tokens, drafts.
//
// Mathematics.  A sequence's queries that share a kv head are rows, token by token, the heads of the group next to each other; a tile has eight.  Products run on the
// tensor cores (m16n8k16, a row to a column: 16 cells or 16 numbers of a value x 8 rows), their 4-bit operand as it lies in the register: masked, n is the f16 n * 2^-24, or n * 2^-20 one
// nibble further up, exactly.
//   scores    with d a block's scale: q . k = sum over blocks b of d_b (sum_i q_i n_i - 8 sum_i q_i).  The sum over i is the product, which starts from what the 8 adds; scales go
//             onto the block's sums in 32 bits.  Numbers of the upper nibble meet queries of a 16th.
//   values    sum over cells of w d_b (n - 8): weights become the other operand transposed (movmatrix), times the scales of their cells, the sum of which times 8 is a product with
//             constants.  The power of two by which weights are larger than exp(score - maximum) follows the largest scale seen, so that neither they nor small products leave f16.
// With F32, queries and weights are two f16 numbers each (22 bits), and the 4-bit operand is made signed (and values scaled, exactly): products of n as it is, up to 15, lose 3e-6 to
// the tensor core's alignment of its 16 terms.  16-bit queries are one f16 number, exactly: a row is scaled by a power of two.
// Softmax by running maximum and sum, per page of 64 cells.
//
// Work.  The pages that a (sequence, tile, kv head) sees, all of them in a row, are dealt out to the CTAs in equal shares, so that lengths do not matter; a CTA's warps take the
// pages of its share in turns, each through a ring of its own (one bulk copy per page: a head's chunk is contiguous), and add up an item in shared memory.  An item that
// is cut goes through the workspace: the CTA that comes last adds the parts in their order (no atomics on numbers, equal calls give equal bits).  Where items have fewer pages than a
// CTA has warps, a warp takes whole items.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cfloat>
#include <type_traits>

#include "../../include/prima_b200.h"
#include "kv4_attn.cuh"

namespace pb {
namespace {

constexpr int KR_WARPS = 12, KR_THREADS = 32 * KR_WARPS, KR_ROWS = 8;
template <int D> constexpr int kr_stages() { return D == 128 ? 2 : 4; }
constexpr int KR_UP = 12;   // F32: weights are 2^12 larger than exp(score - maximum): those of 2^-26 are normal f16 numbers

// what a warp hands to its CTA, a CTA to the last one: sums of 2^(score - m) v, and of the weights
template <int D> struct KrPart { float o[KR_ROWS][D + 4]; float m[KR_ROWS], l[KR_ROWS]; };
static_assert(sizeof(KrPart<128>) <= kv4_chunk_bytes(128) && sizeof(KrPart<64>) <= kv4_chunk_bytes(64), "a warp's part goes through its ring");

template <int D> struct __align__(128) KrSmem {
    __align__(128) uint8_t ring[KR_WARPS][kr_stages<D>()][kv4_chunk_bytes(D)];
    uint64_t full[KR_WARPS][kr_stages<D>()];
    long long scan[KR_WARPS], items[KR_WARPS], before[KR_WARPS];
    KrPart<D> * part[KR_WARPS];
    int seq[KR_WARPS];
    int last, abort;
};

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816_from(float (&d)[4], float c0, float c1, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {   // columns start at c0, c1
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %10, %11};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ void fma2(float & x, float & y, float a, float b, float d) {   // x += a d, y += b d
    asm("{\n.reg .b64 p, q, r;\nmov.b64 p, {%0, %1};\nmov.b64 q, {%2, %3};\nmov.b64 r, {%4, %4};\nfma.rn.f32x2 p, q, r, p;\nmov.b64 {%0, %1}, p;\n}" : "+f"(x), "+f"(y) : "f"(a), "f"(b), "f"(d));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t h2u(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
__device__ __forceinline__ __half2 u2h(uint32_t u) { return *reinterpret_cast<__half2 *>(&u); }

template <typename T, int D>
__global__ void __launch_bounds__(KR_THREADS, 1) k_kv4_attn_rows(const __grid_constant__ Kv4Attn A, const __grid_constant__ KrWork W) {
    constexpr int NB = D / 32, STAGES = kr_stages<D>(), CHUNK = kv4_chunk_bytes(D);
    constexpr bool F32 = std::is_same<T, float>::value;
    constexpr int LO = F32 ? 2 : 1;
    extern __shared__ uint8_t smem_raw[];
    KrSmem<D> & S = *reinterpret_cast<KrSmem<D> *>(smem_raw + ((128u - (smem_u32(smem_raw) & 127u)) & 127u));
    const int tid = threadIdx.x, warp = uniform_warp(), lane = tid & 31, g = lane >> 2, c = lane & 3;
    volatile int * cta_abort = &S.abort;
    if (tid < KR_WARPS * STAGES) mbar_init(&S.full[tid / STAGES][tid % STAGES], 1);
    if (tid == 0) { mbar_fence_init(); S.abort = 0; }

    // ---- shares: units (pages of items) in the order of sequences, tiles, heads, pages ----
    const int hks = A.cache.n_head_kv;
    long long units = 0, items = 0, n = 0;     // n: of this thread's last sequence
    for (int s = tid; s < A.n_seq; s += KR_THREADS) {
        const Kv4Seq q = kv4_seq(A, s, W.most_rows, false);
        n = q.units(hks, KR_ROWS);
        units += n;
        items += q.items(hks, KR_ROWS);
    }
    long long x = units;                       // sums over the lanes up to this one
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
        items += __shfl_xor_sync(0xffffffffu, items, o);
    }
    if (lane == 31) S.scan[warp] = x;
    if (lane == 0) S.items[warp] = items;
    __syncthreads();
    long long total = 0, n_items = 0, front = 0;
#pragma unroll
    for (int w = 0; w < KR_WARPS; w++) {
        if (w < warp) front += S.scan[w];
        total += S.scan[w];
        n_items += S.items[w];
    }
    if (total == 0) return;
    const bool by_warp = total < n_items * KR_WARPS;    // fewer pages an item than a CTA has warps
    const long long among = by_warp ? (long long) gridDim.x * KR_WARPS : (long long) gridDim.x;
    long long share = (total + among - 1) / among;
    if (!by_warp && share < KR_WARPS) share = KR_WARPS;
    // the sequences in which the shares begin
    const long long cta0 = (long long) blockIdx.x * (by_warp ? KR_WARPS : 1) * share;
    auto begins = [&](int s, long long before, long long n) {
#pragma unroll 1
        for (int w = 0; w < (by_warp ? KR_WARPS : 1); w++) {
            const long long u = cta0 + w * share;
            if (u >= before && u < before + n) { S.seq[w] = s; S.before[w] = before; }
        }
    };
    if (A.n_seq <= KR_THREADS) begins(tid, front + x - units, units);
    else {
        long long before = 0;
        for (int s0 = 0; s0 < A.n_seq; s0 += KR_THREADS) {
            n = kv4_seq(A, s0 + tid, W.most_rows, false).units(hks, KR_ROWS);
            x = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            __syncthreads();
            if (lane == 31) S.scan[warp] = x;
            __syncthreads();
            front = before;
            for (int w = 0; w < KR_WARPS; w++) {
                if (w < warp) front += S.scan[w];
                before += S.scan[w];
            }
            begins(s0 + tid, front + x - n, n);
        }
    }
    __syncthreads();
    const long long u0 = cta0 + (by_warp ? warp * share : 0), u1 = u0 + share < total ? u0 + share : total;

    // a place in the row of units: sequence, its first unit, the unit
    struct Place { long long u, before; int s; Kv4Seq q; };
    auto settle = [&](Place & p) {   // onto a sequence that has unit p.u
        while (p.u < u1 && p.u >= p.before + p.q.units(hks, KR_ROWS)) {
            p.before += p.q.units(hks, KR_ROWS);
            p.s++;
            p.q = kv4_seq(A, p.s, W.most_rows, false);
        }
    };
    Place get{u0, 0, 0, {}};
    if (u0 < u1) {
        get.s = S.seq[by_warp ? warp : 0];
        get.before = S.before[by_warp ? warp : 0];
        get.q = kv4_seq(A, get.s, W.most_rows, false);
    }
    if (by_warp && u0 < u1) {   // whole items: those that begin in the share
        const long long in = get.u - get.before;
        const long long r = in % get.q.pages;
        if (r) get.u += get.q.pages - r;
        settle(get);
    }
    Place put = get;

    // ---- pages on their way: the share's pages go to the warps in turns, of a segment [pa, pb) of an item every step-th from pa + first on ----
    const int step = by_warp ? 1 : KR_WARPS;
    auto first_of = [&](long long u) { return by_warp ? 0 : (warp + KR_WARPS - (int) ((u - u0) % KR_WARPS)) % KR_WARPS; };   // u: the segment's first unit
    uint64_t policy;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    int f_pb = 0, f_page = 0, f_hk = 0;       // the segment that is fetched, the next page of it
    bool f_more = false;
    auto segment = [&](Place & p, int & pa, int & pb, int & tile, int & hk, int & first) {   // false: no more
        if (p.u >= u1) return false;
        settle(p);
        const long long in = p.u - p.before;
        const int item = (int) (in / p.q.pages);
        pa = (int) (in - (long long) item * p.q.pages);
        const long long rest = by_warp ? p.q.pages : u1 - p.u;
        pb = (int) (pa + rest < p.q.pages ? pa + rest : p.q.pages);
        tile = item / hks;
        hk = item % hks;
        first = pa + first_of(p.u);
        p.u += pb - pa;
        return true;
    };
    auto next_page = [&]() {   // page number of the next page of this warp, or -1 (nothing to fetch); moves on
        while (true) {
            if (f_more && f_page < f_pb) {
                const int i = f_page;
                f_page += step;
                return kv4_page(A, get.q, get.s, i);
            }
            int pa, tile;
            f_more = segment(get, pa, f_pb, tile, f_hk, f_page);
            if (!f_more) return -2;
        }
    };
    uint32_t issued = 0, used = 0;                      // pages asked for and taken, of this warp
    int ids[STAGES];                                    // their numbers (-1: none), by stage
    auto fetch = [&]() {
        const int id = next_page();
        const int st = (int) (issued % STAGES);
#pragma unroll
        for (int i = 0; i < STAGES; i++)
            if (i == st) ids[i] = id;
        if (id >= 0 && elect_one()) {
            mbar_arrive_expect_tx(&S.full[warp][st], CHUNK);
            bulk_g2s(S.ring[warp][st], kv4_chunk<D>(A.cache, id, f_hk), CHUNK, &S.full[warp][st], policy);
        }
        __syncwarp();
        issued++;
    };
    uint32_t phases = 0;
    for (int i = 0; i < STAGES; i++) fetch();

    // ---- segments ----
    int pa, pb, tile, hk, first;
    while (segment(put, pa, pb, tile, hk, first)) {
        const Kv4Seq q = put.q;
        const int row0 = tile * KR_ROWS, rows = min(KR_ROWS, q.n_q * A.group - row0);
        // queries: lane (g, c) has of row g the numbers 32 b + 8 c + e, as pairs; F32: two f16 numbers each (high, low), otherwise pairs 1 and 3 a 16th
        uint32_t qf[LO][NB][4];
        float start[NB][2], mult[2];
        int pos[2];
        {
            float x[NB][8];
            const int row = row0 + g;
            const bool have = g < rows;
            const T * src = (const T *) A.q + (q.q0 + row / A.group) * A.ldq + (int64_t) (hk * A.group + row % A.group) * D + 8 * c;
            float top = 0.f;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const float4 lo4 = have ? load4(src + 32 * b) : make_float4(0.f, 0.f, 0.f, 0.f), hi4 = have ? load4(src + 32 * b + 4) : make_float4(0.f, 0.f, 0.f, 0.f);
                x[b][0] = lo4.x; x[b][1] = lo4.y; x[b][2] = lo4.z; x[b][3] = lo4.w;
                x[b][4] = hi4.x; x[b][5] = hi4.y; x[b][6] = hi4.z; x[b][7] = hi4.w;
#pragma unroll
                for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(x[b][e]));
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // the row's power of two: its largest number comes to 2^13 .. 2^14
            const int ex = top > 0.f && top < INFINITY ? max(-126, min(126, 13 - ilogbf(top))) : 0;
            const float up = __int_as_float((ex + 127) << 23) * (A.scale < 0.f ? -1.f : 1.f);
            float sums[NB];
#pragma unroll
            for (int b = 0; b < NB; b++) {
                float sum = 0.f;
#pragma unroll
                for (int p = 0; p < 4; p++) {
                    const float y0 = x[b][2 * p] * up, y1 = x[b][2 * p + 1] * up;
                    sum += y0 + y1;
                    const __half2 h = __floats2half2_rn(y0, y1);
                    if constexpr (F32) {
                        const float2 back = __half22float2(h);
                        qf[0][b][p] = h2u(h);
                        qf[LO - 1][b][p] = h2u(__floats2half2_rn(y0 - back.x, y1 - back.y));
                    } else qf[0][b][p] = h2u(p & 1 ? __hmul2(h, __float2half2_rn(0.0625f)) : h);
                }
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                sums[b] = sum * (-8.f / 16777216.f);
            }
            // of a row's sums: the power of two, n * 2^-24, and scores in units of log2; never 0: a masked score stays -inf
            const float down = fmaxf(fabsf(A.scale) * (F32 ? 1.4426950408889634f : 1.4426950408889634f * 16777216.f) * __int_as_float((127 - ex) << 23), FLT_MIN);
            const int at = q.p0 + row / A.group;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int from = 4 * (2 * c + i);                               // a lane of row 2 c + i
                mult[i] = __shfl_sync(0xffffffffu, down, from);
                pos[i] = __shfl_sync(0xffffffffu, have ? at : -1, from);
#pragma unroll
                for (int b = 0; b < NB; b++) start[b][i] = F32 ? 0.f : __shfl_sync(0xffffffffu, sums[b], from);
            }
        }
        const int p_lo = q.p0 + row0 / A.group, p_hi = q.p0 + (row0 + rows - 1) / A.group;   // of the tile's rows

        // out^T: lane: numbers 32 b + 4 g + 2 h, + 1 of rows 2 c, 2 c + 1; 16 bits: odd numbers 16 times as large, and o8: 8 times the sum of scaled weights (odd: 128 times)
        float o[NB][2][4], o8[F32 ? 1 : NB][4];
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
        int up = F32 ? KR_UP : 15;                      // weights are exp(score - maximum) * 2^up
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                o[b][0][i] = o[b][1][i] = 0.f;
                if constexpr (!F32) o8[b][i] = 0.f;
            }
        bool any = false;
        uint8_t * held = nullptr;                       // the stage of the segment's last page: handed back behind the merge
        for (int i = first; i < pb; i += step) {
            const int st = (int) (used % STAGES);
            int id = -1;
#pragma unroll
            for (int k = 0; k < STAGES; k++)
                if (k == st) id = ids[k];
            used++;
            const bool keep = !by_warp && i + step >= pb;
            if (id >= 0) {
                mbar_wait(&S.full[warp][st], phases >> st & 1, cta_abort, W.abort_flag);
                phases ^= 1u << st;
                uint8_t * chunk = S.ring[warp][st];
                uint8_t * const vs = chunk + 2 * kv4_rows_bytes(D) + kv4_scales_bytes(D);
                const int base = kv4_page_index(q, i) * KV4_CELLS;
                const bool whole = base + 63 <= p_lo && (A.window <= 0 || p_hi - base < A.window || base + 63 < A.first);
                if (!whole) {   // a weight of zero does not silence a scale that is no number: cells nobody sees may hold anything
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int t = 2 * lane + e, cell = base + t;
                        if (!(cell <= p_hi && (A.window <= 0 || p_lo - cell < A.window || cell < A.first)))
#pragma unroll
                            for (int b = 0; b < NB; b++) *reinterpret_cast<uint16_t *>(vs + kv4_scale(D, t, b)) = 0;
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // ahead of the copy that takes this stage next
                    __syncwarp();
                }
                // scores: 16 cells at a time; lane: cells 16 j + g, 16 j + 8 + g of rows 2 c, 2 c + 1
                float sc[4][4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    uint32_t wa[NB], wb[NB];
                    const uint8_t * ra = chunk + (16 * j + g) * (D / 2) + 4 * NB * c, * rb = ra + 8 * (D / 2);
                    if constexpr (NB == 4) {
                        *reinterpret_cast<uint4 *>(wa) = *reinterpret_cast<const uint4 *>(ra);
                        *reinterpret_cast<uint4 *>(wb) = *reinterpret_cast<const uint4 *>(rb);
                    } else {
                        *reinterpret_cast<uint2 *>(wa) = *reinterpret_cast<const uint2 *>(ra);
                        *reinterpret_cast<uint2 *>(wb) = *reinterpret_cast<const uint2 *>(rb);
                    }
                    const uint8_t * ks = chunk + 2 * kv4_rows_bytes(D) + kv4_scale(D, 16 * j + g, 0);
#pragma unroll
                    for (int i4 = 0; i4 < 4; i4++) sc[j][i4] = 0.f;
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        float acc[4];
                        const uint32_t a1 = wa[b] >> 8, b1 = wb[b] >> 8;
                        if constexpr (F32) {
                            auto even = [](uint32_t w) { return h2u(__hsub2(u2h((w & 0x000f000fu) | 0x64006400u), __float2half2_rn(1032.f))); };   // 1024 + n
                            auto odd = [](uint32_t w) { return h2u(__hsub2(u2h((w & 0x00f000f0u) | 0x54005400u), __float2half2_rn(72.f))); };      // 64 + n
                            const uint32_t x[8] = {even(wa[b]), even(wb[b]), odd(wa[b]), odd(wb[b]), even(a1), even(b1), odd(a1), odd(b1)};
                            mma16816_from(acc, 0.f, 0.f, x[0], x[1], x[2], x[3], qf[0][b][0], qf[0][b][1]);
                            mma16816(acc, x[4], x[5], x[6], x[7], qf[0][b][2], qf[0][b][3]);
                            mma16816(acc, x[0], x[1], x[2], x[3], qf[LO - 1][b][0], qf[LO - 1][b][1]);
                            mma16816(acc, x[4], x[5], x[6], x[7], qf[LO - 1][b][2], qf[LO - 1][b][3]);
                        } else {
                            mma16816_from(acc, start[b][0], start[b][1], wa[b] & 0x000f000fu, wb[b] & 0x000f000fu, wa[b] & 0x00f000f0u, wb[b] & 0x00f000f0u, qf[0][b][0], qf[0][b][1]);
                            mma16816(acc, a1 & 0x000f000fu, b1 & 0x000f000fu, a1 & 0x00f000f0u, b1 & 0x00f000f0u, qf[0][b][2], qf[0][b][3]);
                        }
                        fma2(sc[j][0], sc[j][1], acc[0], acc[1], __half2float(*reinterpret_cast<const __half *>(ks + 4 * b)));
                        fma2(sc[j][2], sc[j][3], acc[2], acc[3], __half2float(*reinterpret_cast<const __half *>(ks + 4 * b + 16 * NB)));
                    }
                }
                if (!whole) {
#pragma unroll
                    for (int j = 0; j < 4; j++)
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const int cell = base + 16 * j + g + (k >> 1) * 8, p = pos[k & 1];
                            if (!(cell <= p && (A.window <= 0 || p - cell < A.window || cell < A.first))) sc[j][k] = -INFINITY;
                        }
                }
                float mx[2];
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    float a = fmaxf(fmaxf(sc[0][k], sc[0][k + 2]), fmaxf(sc[1][k], sc[1][k + 2])), b = fmaxf(fmaxf(sc[2][k], sc[2][k + 2]), fmaxf(sc[3][k], sc[3][k + 2]));
                    a = fmaxf(a, b);
                    a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 4));
                    a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 8));
                    a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 16));
                    mx[k] = a * mult[k];
                }
                int to = up;
                if constexpr (!F32) {   // lane: the scales of cells 2 lane, 2 lane + 1
                    uint32_t w[NB], top = 0;
                    const uint8_t * src = vs + 4 * NB * lane;
                    if constexpr (NB == 4) *reinterpret_cast<uint4 *>(w) = *reinterpret_cast<const uint4 *>(src);
                    else *reinterpret_cast<uint2 *>(w) = *reinterpret_cast<const uint2 *>(src);
#pragma unroll
                    for (int b = 0; b < NB; b++) top = __vmaxu2(top, w[b] & 0x7fff7fffu);
                    top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));
                    to = min(up, 29 - (int) (top >> 10));   // the largest scale is below 2^(top / 1024 - 14): products stay below 2^15
                }
                if (__any_sync(0xffffffffu, mx[0] > m[0] || mx[1] > m[1]) || to != up) {
                    float f[2];
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        const float mn = fmaxf(m[k], mx[k]);
                        f[k] = m[k] == -INFINITY ? 0.f : ex2(m[k] - mn + (float) (to - up));
                        m[k] = mn;
                        l[k] *= f[k];
                    }
                    up = to;
#pragma unroll
                    for (int b = 0; b < NB; b++) {
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            o[b][h][0] *= f[0]; o[b][h][1] *= f[1];
                            o[b][h][2] *= f[0]; o[b][h][3] *= f[1];
                        }
                        if constexpr (!F32) {
                            o8[b][0] *= f[0]; o8[b][1] *= f[1];
                            o8[b][2] *= f[0]; o8[b][3] *= f[1];
                        }
                    }
                }
                const float off[2] = {m[0] == -INFINITY ? 0.f : (float) up - m[0], m[1] == -INFINITY ? 0.f : (float) up - m[1]};
                // weights, transposed: lane: row g, cells 8 x + 2 c, + 1 (x: eights of the page)
                uint32_t pf[LO][8];
#pragma unroll
                for (int x8 = 0; x8 < 8; x8++) {
                    const float e0 = ex2(fmaf(sc[x8 >> 1][2 * (x8 & 1)], mult[0], off[0])), e1 = ex2(fmaf(sc[x8 >> 1][2 * (x8 & 1) + 1], mult[1], off[1]));
                    fma2(l[0], l[1], e0, e1, 1.f);
                    const __half2 h = __floats2half2_rn(e0, e1);
                    pf[0][x8] = transposed(h2u(h));
                    if constexpr (F32) {
                        const float2 back = __half22float2(h);
                        pf[LO - 1][x8] = transposed(h2u(__floats2half2_rn(e0 - back.x, e1 - back.y)));
                    }
                }
                // values: lane: numbers 32 b + 4 g + i of cells 16 j + 2 c, + 1 and 16 j + 8 + 2 c, + 1
                const uint8_t * vr = chunk + kv4_rows_bytes(D) + c * (D / 2) + 2 * NB * (g ^ (4 * ((c >> 1) & 1)));
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    uint32_t w[4][NB / 2], d[2][NB];   // cells 2c, 2c+1, 8+2c, 9+2c
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint8_t * src = vr + (16 * j + 8 * (k >> 1) + 4 * (k & 1)) * (D / 2);      // row of the cell
                        if constexpr (NB == 4) *reinterpret_cast<uint2 *>(w[k]) = *reinterpret_cast<const uint2 *>(src);
                        else w[k][0] = *reinterpret_cast<const uint32_t *>(src);
                    }
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        const uint8_t * src = vs + kv4_scale(D, 16 * j + 8 * k + 2 * c, 0);
                        if constexpr (NB == 4) *reinterpret_cast<uint4 *>(d[k]) = *reinterpret_cast<const uint4 *>(src);
                        else *reinterpret_cast<uint2 *>(d[k]) = *reinterpret_cast<const uint2 *>(src);
                    }
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        uint32_t u[2];   // of an eight: numbers of the two cells
#pragma unroll
                        for (int k = 0; k < 2; k++) u[k] = __byte_perm(w[2 * k][b / 2], w[2 * k + 1][b / 2], b & 1 ? 0x7632 : 0x5410);
                        if constexpr (F32) {
                            uint32_t v[2][4];
#pragma unroll
                            for (int k = 0; k < 2; k++) {
                                const __half2 sd = u2h(d[k][b]), s24 = __hmul2(sd, __float2half2_rn(-24.f));
                                v[k][0] = h2u(__hmul2(__hsub2(u2h((u[k] & 0x000f000fu) | 0x64006400u), __float2half2_rn(1032.f)), sd));                // 1024 + n
                                v[k][1] = h2u(__hmul2(__hsub2(u2h((u[k] & 0x00f000f0u) | 0x54005400u), __float2half2_rn(72.f)), sd));                  // 64 + n
                                v[k][2] = h2u(__hfma2(u2h((u[k] >> 2 & 0x03c003c0u) | 0x4c004c00u), sd, s24));                                         // 16 + n: 24 scales are an f16
                                v[k][3] = h2u(__hfma2(u2h((u[k] >> 6 & 0x03c003c0u) | 0x4c004c00u), sd, s24));
                            }
#pragma unroll
                            for (int h = 0; h < LO; h++) {
                                mma16816(o[b][0], v[0][0], v[0][1], v[1][0], v[1][1], pf[h][2 * j], pf[h][2 * j + 1]);
                                mma16816(o[b][1], v[0][2], v[0][3], v[1][2], v[1][3], pf[h][2 * j], pf[h][2 * j + 1]);
                            }
                        } else {
                            const uint32_t p0 = h2u(__hmul2(u2h(pf[0][2 * j]), u2h(d[0][b]))), p1 = h2u(__hmul2(u2h(pf[0][2 * j + 1]), u2h(d[1][b])));
                            const uint32_t s0 = u[0] >> 8, s1 = u[1] >> 8;
                            mma16816(o[b][0], u[0] & 0x000f000fu, u[0] & 0x00f000f0u, u[1] & 0x000f000fu, u[1] & 0x00f000f0u, p0, p1);
                            mma16816(o[b][1], s0 & 0x000f000fu, s0 & 0x00f000f0u, s1 & 0x000f000fu, s1 & 0x00f000f0u, p0, p1);
                            mma16816(o8[b], 0x00080008u, 0x00800080u, 0x00080008u, 0x00800080u, p0, p1);
                        }
                    }
                }
                any = true;
            }
            if (!keep) {
                __syncwarp();
                fetch();
            } else held = S.ring[warp][st];
        }
#pragma unroll
        for (int k = 0; k < 2; k++) {
            l[k] += __shfl_xor_sync(0xffffffffu, l[k], 4);
            l[k] += __shfl_xor_sync(0xffffffffu, l[k], 8);
            l[k] += __shfl_xor_sync(0xffffffffu, l[k], 16);
        }
        if constexpr (!F32)
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int i = 0; i < 4; i++) o[b][h][i] = (o[b][h][i] - o8[b][i]) * (i < 2 ? 16777216.f : 1048576.f);
        T * out = (T *) A.out + (int64_t) hk * A.group * D;
        auto row_of = [&](int r) { return out + (q.q0 + (row0 + r) / A.group) * A.ldo + (int64_t) ((row0 + r) % A.group) * D; };
        if (by_warp) {
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const int r = 2 * c + k;
                const float inv = l[k] == 0.f ? 0.f : 1.f / l[k];
                if (r < rows)
#pragma unroll
                    for (int b = 0; b < NB; b++)
                        store4(row_of(r) + 32 * b + 4 * g, make_float4(o[b][0][k] * inv, o[b][0][2 + k] * inv, o[b][1][k] * inv, o[b][1][2 + k] * inv));
            }
            continue;
        }
        // ---- the CTA's sum ----
        KrPart<D> * part = reinterpret_cast<KrPart<D> *>(held);
        if (any) {
            __syncwarp();
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const int r = 2 * c + k;
#pragma unroll
                for (int b = 0; b < NB; b++) *reinterpret_cast<float4 *>(&part->o[r][32 * b + 4 * g]) = make_float4(o[b][0][k], o[b][0][2 + k], o[b][1][k], o[b][1][2 + k]);
                if (g == 0) { part->m[r] = m[k] - (float) up; part->l[r] = l[k]; }
            }
        }
        if (lane == 0) S.part[warp] = any ? part : nullptr;
        __syncthreads();
        const bool full = pa == 0 && pb == q.pages;
        KrPart<D> * ws = reinterpret_cast<KrPart<D> *>(W.parts);
        KrPart<D> * to = &ws[2 * blockIdx.x + (pa > 0 ? 0 : 1)];
        const int r = tid / (D / 4), d4 = 4 * (tid % (D / 4));
        auto write = [&](float4 x, float sum) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            if (r < rows) store4(row_of(r) + d4, make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
        };
        // parts in their order: at(i) is one, or none
        float top = -INFINITY, sum = 0.f;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        auto add = [&](float mi, float li, float4 y) {
            const float tn = fmaxf(top, mi);
            const float f = top == -INFINITY ? (sum == sum ? 0.f : 1.f) : ex2(top - tn), h = mi == -INFINITY ? (li == li ? 0.f : 1.f) : ex2(mi - tn);
            top = tn;
            sum = sum * f + li * h;
            x.x = x.x * f + y.x * h; x.y = x.y * f + y.y * h; x.z = x.z * f + y.z * h; x.w = x.w * f + y.w * h;
        };
        if (r < KR_ROWS) {
#pragma unroll 2
            for (int i = 0; i < KR_WARPS; i++)
                if (const KrPart<D> * p = S.part[i]) add(p->m[r], p->l[r], *reinterpret_cast<const float4 *>(&p->o[r][d4]));
            if (full) write(x, sum);
            else {
                *reinterpret_cast<float4 *>(&to->o[r][d4]) = x;
                if (d4 == 0) { to->m[r] = top; to->l[r] = sum; }
            }
        }
        if (!full) {
            const long long a0 = put.before + (long long) (tile * hks + hk) * q.pages;                     // the item's first unit
            const int c0 = (int) (a0 / share), n_parts = (int) ((a0 + q.pages - 1) / share) - c0 + 1;       // the CTAs that share it
            __threadfence();
            __syncthreads();
            if (tid == 0) S.last = atomicAdd(&W.counters[c0], 1) == n_parts - 1;
            __syncthreads();
            if (S.last) {
                __threadfence();
                if (r < KR_ROWS) {
                    top = -INFINITY; sum = 0.f; x = make_float4(0.f, 0.f, 0.f, 0.f);
                    constexpr int AT_ONCE = 8;                       // on their way from L2 together
                    for (int i0 = 0; i0 < n_parts; i0 += AT_ONCE) {
                        float mi[AT_ONCE], li[AT_ONCE];
                        float4 y[AT_ONCE];
#pragma unroll
                        for (int k = 0; k < AT_ONCE; k++) {
                            const int i = min(i0 + k, n_parts - 1);
                            const KrPart<D> * p = &ws[2 * (c0 + i) + (i == 0 ? 1 : 0)];
                            mi[k] = __ldcg(&p->m[r]);
                            li[k] = __ldcg(&p->l[r]);
                            y[k] = __ldcg(reinterpret_cast<const float4 *>(&p->o[r][d4]));
                        }
#pragma unroll
                        for (int k = 0; k < AT_ONCE; k++)
                            if (i0 + k < n_parts) add(mi[k], li[k], y[k]);
                    }
                    write(x, sum);
                }
                if (tid == 0) W.counters[c0] = 0;
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // what was read and written of a stage, the next copy overwrites
        __syncthreads();
        if (held) fetch();
    }
}

template <typename T, int D>
int rows_launch(const Kv4Attn & a, const KrWork & w, cudaStream_t st) {
    constexpr size_t smem = sizeof(KrSmem<D>) + 128;
    static_assert(smem <= 232448, "shared memory of an SM");
    static FuncAttrCache cache;
    const cudaError_t e = ensure_dyn_smem(cache, (const void *) k_kv4_attn_rows<T, D>, smem, true);
    if (e != cudaSuccess) return (int) e;
    k_kv4_attn_rows<T, D><<<sm_count() < KV4_MAX_CTAS ? sm_count() : KV4_MAX_CTAS, KR_THREADS, smem, st>>>(a, w);
    return (int) cudaGetLastError();
}

}  // namespace

size_t kv4_rows_workspace(int D) { return 2 * (size_t) KV4_MAX_CTAS * (D == 128 ? sizeof(KrPart<128>) : sizeof(KrPart<64>)); }

int launch_kv4_attn_rows(const Kv4Attn & a, int D, int type, int most_rows, int * counters, void * parts, cudaStream_t st) {
    const KrWork w{most_rows, counters, parts, abort_flag()};
    if (D == 128) return type == PB200_TYPE_F32 ? rows_launch<float, 128>(a, w, st) : type == PB200_TYPE_F16 ? rows_launch<__half, 128>(a, w, st) : rows_launch<__nv_bfloat16, 128>(a, w, st);
    return type == PB200_TYPE_F32 ? rows_launch<float, 64>(a, w, st) : type == PB200_TYPE_F16 ? rows_launch<__half, 64>(a, w, st) : rows_launch<__nv_bfloat16, 64>(a, w, st);
}

}  // namespace pb
