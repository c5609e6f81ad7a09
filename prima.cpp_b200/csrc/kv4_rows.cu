// prima.cpp_b200/csrc/kv4_rows.cu — attention over the 4-bit cache (kv4.cuh) for sequences with few query rows: single tokens, drafts.
//
// Mathematics.  A sequence's queries that share a kv head are rows, token by token, the heads of the group next to each other; a tile has eight.  With n the 4 bits of a key's
// number, d its block's scale: q . k = sum over blocks b of d_b (sum_i q_i n_i - 8 sum_i q_i).  The inner sum runs on the tensor cores (m16n8k16: 16 cells x 8 rows), on n as it
// lies in the register: masked, it is the f16 n * 2^-24 (or 2^-20, against queries of a 16th), exactly; what the 8 adds is where the sum starts.  Scales are applied to the
// block's 16 x 8 sums in 32 bits.  Values become f16 numbers, exactly, and weights' transposes (movmatrix) are the other operand: out^T (16 numbers x 8 rows) += V^T P^T.  With
// F32, queries and weights are two f16 numbers each (22 bits); 16-bit queries are one, exactly (a row is scaled by a power of two), and weights one.
// Softmax by running maximum and sum, per page of 64 cells.
//
// Work.  The pages that a (sequence, tile, kv head) sees, all of them in a row, are dealt out to the CTAs in equal shares, so that lengths do not matter; a CTA's warps take the
// pages of an item in turns, each through a ring of its own (one bulk copy per page: a head's chunk is contiguous), and add up in shared memory.  An item that
// is cut goes through the workspace: the CTA that comes last adds the parts in their order (no atomics on numbers, equal calls give equal bits).  Where items have fewer pages than a
// CTA has warps, a warp takes whole items.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "../../include/prima_b200.h"
#include "kv4_attn.cuh"

namespace pb {
namespace {

constexpr int KR_WARPS = 12, KR_THREADS = 32 * KR_WARPS, KR_ROWS = 8;
template <int D> constexpr int kr_stages() { return D == 128 ? 2 : 4; }
constexpr float KR_UP = 12.f;   // weights are 2^12 larger than exp(score - maximum): those of 2^-26 are normal f16 numbers

template <int D> struct KrPart { float o[KR_ROWS][D + 4]; float m[KR_ROWS], l[KR_ROWS]; };   // what a warp hands to its CTA, a CTA to the last one
static_assert(sizeof(KrPart<128>) <= kv4_chunk_bytes(128) && sizeof(KrPart<64>) <= kv4_chunk_bytes(64), "a warp's part goes through its ring");

template <int D> struct __align__(128) KrSmem {
    __align__(128) uint8_t ring[KR_WARPS][kr_stages<D>()][kv4_chunk_bytes(D)];
    uint64_t full[KR_WARPS][kr_stages<D>()];
    long long scan[KR_WARPS], items[KR_WARPS];
    KrPart<D> * part[KR_WARPS];
    int last, abort;
};

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t h2u(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
__device__ __forceinline__ __half2 u2h(uint32_t u) { return *reinterpret_cast<__half2 *>(&u); }

// One page's walk.  Everything here is the same for all lanes of a warp.
struct KrItem { int s, hk, row0, rows, n_q; int64_t q0; int p0; };   // p0: position of the sequence's first query

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
    long long units = 0, items = 0;
    for (int s = tid; s < A.n_seq; s += KR_THREADS) {
        const Kv4Seq q = kv4_seq(A, s, W.most_rows, false);
        units += q.units(A.cache.n_head_kv, KR_ROWS);
        items += q.items(A.cache.n_head_kv, KR_ROWS);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        units += __shfl_xor_sync(0xffffffffu, units, o);
        items += __shfl_xor_sync(0xffffffffu, items, o);
    }
    if (lane == 0) { S.scan[warp] = units; S.items[warp] = items; }
    __syncthreads();
    long long total = 0, n_items = 0;
    for (int w = 0; w < KR_WARPS; w++) {
        total += S.scan[w];
        n_items += S.items[w];
    }
    if (total == 0) return;
    const bool by_warp = total < n_items * KR_WARPS;    // fewer pages an item than a CTA has warps
    long long share = (total + gridDim.x - 1) / gridDim.x;
    if (share < KR_WARPS) share = KR_WARPS;
    if (by_warp) share = (total + (long long) gridDim.x * KR_WARPS - 1) / ((long long) gridDim.x * KR_WARPS);
    const long long me = by_warp ? (long long) blockIdx.x * KR_WARPS + warp : blockIdx.x;
    const long long u0 = me * share, u1 = u0 + share < total ? u0 + share : total;

    // the sequence that holds unit u, and the units in front of it: a walk over the sequences, 32 at a time
    auto find = [&](long long u, int & seq, long long & before) {
        before = 0;
        for (int s0 = 0; s0 < A.n_seq; s0 += 32) {
            const int s = s0 + lane;
            const long long n = s < A.n_seq ? kv4_seq(A, s, W.most_rows, false).units(A.cache.n_head_kv, KR_ROWS) : 0;
            long long x = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            const uint32_t in = __ballot_sync(0xffffffffu, u < before + x);
            if (in) {
                const int at = __ffs((int) in) - 1;
                seq = s0 + at;
                before += __shfl_sync(0xffffffffu, x - n, at);
                return;
            }
            before += __shfl_sync(0xffffffffu, x, 31);
        }
        seq = A.n_seq;
    };

    // a place in the row of units: sequence, its first unit, the unit
    struct Place { long long u, before; int s; Kv4Seq q; };
    auto settle = [&](Place & p) {   // onto a sequence that has unit p.u
        while (p.u < u1 && p.u >= p.before + p.q.units(A.cache.n_head_kv, KR_ROWS)) {
            p.before += p.q.units(A.cache.n_head_kv, KR_ROWS);
            p.s++;
            p.q = kv4_seq(A, p.s, W.most_rows, false);
        }
    };
    Place get{u0, 0, 0, {}};
    if (u0 < u1) {
        find(u0, get.s, get.before);
        get.q = kv4_seq(A, get.s, W.most_rows, false);
    }
    if (by_warp && u0 < u1) {   // whole items: those that begin in the share
        const long long in = get.u - get.before;
        const long long r = in % get.q.pages;
        if (r) get.u += get.q.pages - r;
        settle(get);
    }
    Place put = get;

    // ---- pages on their way: of a segment [pa, pb) of an item, this warp's are pa + first, pa + first + step, ... ----
    const int first = by_warp ? 0 : warp, step = by_warp ? 1 : KR_WARPS;
    uint64_t policy;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    int f_pa = 0, f_pb = 0, f_page = 0, f_hk = 0;       // the segment that is fetched, the next page of it
    bool f_more = false;
    auto segment = [&](Place & p, int & pa, int & pb, int & tile, int & hk) {   // false: no more
        if (p.u >= u1) return false;
        settle(p);
        const long long in = p.u - p.before;
        const int item = (int) (in / p.q.pages);
        pa = (int) (in - (long long) item * p.q.pages);
        const long long rest = by_warp ? p.q.pages : u1 - p.u;
        pb = (int) (pa + rest < p.q.pages ? pa + rest : p.q.pages);
        tile = item / A.cache.n_head_kv;
        hk = item % A.cache.n_head_kv;
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
            int tile;
            f_more = segment(get, f_pa, f_pb, tile, f_hk);
            if (!f_more) return -2;
            f_page = f_pa + first;
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
    __syncthreads();
    uint32_t phases = 0;
    for (int i = 0; i < STAGES; i++) fetch();

    // ---- segments ----
    int pa, pb, tile, hk;
    while (segment(put, pa, pb, tile, hk)) {
        const Kv4Seq q = put.q;
        const int s = put.s, row0 = tile * KR_ROWS, rows = min(KR_ROWS, q.n_q * A.group - row0);
        // queries: lane (g, c) has of row g the numbers 32 b + 8 c + e; two f16 numbers (high, low) each of pairs 2p, 2p+1, pairs 1 and 3 by a 16th
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
            const float up = __int_as_float((ex + 127) << 23);
            float sums[NB];
#pragma unroll
            for (int b = 0; b < NB; b++) {
                float sum = 0.f;
#pragma unroll
                for (int p = 0; p < 4; p++) {
                    const float y0 = x[b][2 * p] * up, y1 = x[b][2 * p + 1] * up;
                    sum += y0 + y1;
                    const __half2 h = __floats2half2_rn(y0, y1);
                    const __half2 f = __float2half2_rn(p & 1 ? 0.0625f : 1.f);
                    qf[0][b][p] = h2u(__hmul2(h, f));
                    if constexpr (F32) {
                        const float2 back = __half22float2(h);
                        qf[LO - 1][b][p] = h2u(__hmul2(__floats2half2_rn(y0 - back.x, y1 - back.y), f));
                    }
                }
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                sums[b] = sum * (-8.f / 16777216.f);
            }
            const float back = A.scale * 1.4426950408889634f * 16777216.f;      // of a row's sums: the power of two, n * 2^-24, and scores in units of log2
            const float down = back * __int_as_float((127 - ex) << 23);
            const int at = q.p0 + row / A.group;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int from = 4 * (2 * c + i);                               // a lane of row 2 c + i
                mult[i] = __shfl_sync(0xffffffffu, down, from);
                pos[i] = __shfl_sync(0xffffffffu, have ? at : -1, from);
#pragma unroll
                for (int b = 0; b < NB; b++) start[b][i] = __shfl_sync(0xffffffffu, sums[b], from);
            }
        }
        const int p_lo = q.p0 + row0 / A.group, p_hi = q.p0 + (row0 + rows - 1) / A.group;   // of the tile's rows

        float o[NB][2][4];
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int i = 0; i < 4; i++) o[b][h][i] = 0.f;
        bool any = false;
        uint8_t * held = nullptr;                       // the stage of the segment's last page: handed back behind the merge
        for (int i = pa + first; i < pb; i += step) {
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
                const uint8_t * chunk = S.ring[warp][st];
                const int base = kv4_page_index(q, i) * KV4_CELLS;
                const bool whole = base + 63 <= p_lo && (A.window <= 0 || p_hi - base < A.window || base + 63 < A.first);
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
                        float acc[4] = {start[b][0], start[b][1], start[b][0], start[b][1]};
                        const uint32_t a1 = wa[b] >> 8, b1 = wb[b] >> 8;
#pragma unroll
                        for (int h = 0; h < LO; h++) {
                            mma16816(acc, wa[b] & 0x000f000fu, wb[b] & 0x000f000fu, wa[b] & 0x00f000f0u, wb[b] & 0x00f000f0u, qf[h][b][0], qf[h][b][1]);
                            mma16816(acc, a1 & 0x000f000fu, b1 & 0x000f000fu, a1 & 0x00f000f0u, b1 & 0x00f000f0u, qf[h][b][2], qf[h][b][3]);
                        }
                        const float da = __half2float(*reinterpret_cast<const __half *>(ks + 4 * b)), db = __half2float(*reinterpret_cast<const __half *>(ks + 4 * b + 16 * NB));
                        sc[j][0] = fmaf(acc[0], da, sc[j][0]);
                        sc[j][1] = fmaf(acc[1], da, sc[j][1]);
                        sc[j][2] = fmaf(acc[2], db, sc[j][2]);
                        sc[j][3] = fmaf(acc[3], db, sc[j][3]);
                    }
                }
                float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        float t = sc[j][k] * mult[k & 1];
                        if (!whole) {
                            const int cell = base + 16 * j + g + (k >> 1) * 8, p = pos[k & 1];
                            const bool see = cell <= p && (A.window <= 0 || p - cell < A.window || cell < A.first);
                            t = see ? t : -INFINITY;
                        }
                        sc[j][k] = t;
                        mx[k & 1] = fmaxf(mx[k & 1], t);
                    }
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    mx[k] = fmaxf(mx[k], __shfl_xor_sync(0xffffffffu, mx[k], 4));
                    mx[k] = fmaxf(mx[k], __shfl_xor_sync(0xffffffffu, mx[k], 8));
                    mx[k] = fmaxf(mx[k], __shfl_xor_sync(0xffffffffu, mx[k], 16));
                }
                if (__any_sync(0xffffffffu, mx[0] > m[0] || mx[1] > m[1])) {
                    float f[2];
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        const float mn = fmaxf(m[k], mx[k]);
                        f[k] = m[k] == -INFINITY ? 0.f : ex2(m[k] - mn);
                        m[k] = mn;
                        l[k] *= f[k];
                    }
#pragma unroll
                    for (int b = 0; b < NB; b++)
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            o[b][h][0] *= f[0]; o[b][h][1] *= f[1];
                            o[b][h][2] *= f[0]; o[b][h][3] *= f[1];
                        }
                }
                const float off[2] = {m[0] == -INFINITY ? 0.f : m[0] - KR_UP, m[1] == -INFINITY ? 0.f : m[1] - KR_UP};
                // weights, transposed: lane: row g, cells 8 x + 2 c, + 1 (x: eights of the page)
                uint32_t pf[LO][8];
#pragma unroll
                for (int x = 0; x < 8; x++) {
                    const float e0 = ex2(sc[x >> 1][2 * (x & 1)] - off[0]), e1 = ex2(sc[x >> 1][2 * (x & 1) + 1] - off[1]);
                    l[0] += e0;
                    l[1] += e1;
                    const __half2 h = __floats2half2_rn(e0, e1);
                    pf[0][x] = transposed(h2u(h));
                    if constexpr (F32) {
                        const float2 back = __half22float2(h);
                        pf[LO - 1][x] = transposed(h2u(__floats2half2_rn(e0 - back.x, e1 - back.y)));
                    }
                }
                // values: lane: numbers 32 b + 4 g + i of cells 16 j + 2 c, + 1 and 16 j + 8 + 2 c, + 1
                const uint8_t * vr = chunk + kv4_rows_bytes(D);
                const uint8_t * vs = chunk + 2 * kv4_rows_bytes(D) + kv4_scales_bytes(D);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    uint32_t w[4][NB / 2], d[2][NB];   // cells 2c, 2c+1, 8+2c, 9+2c
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const int r = 16 * j + 8 * (k >> 1) + 4 * (k & 1) + c;                   // row of the cell
                        const uint8_t * src = vr + r * (D / 2) + 2 * NB * (g ^ (4 * ((c >> 1) & 1)));
                        if constexpr (NB == 4) *reinterpret_cast<uint2 *>(w[k]) = *reinterpret_cast<const uint2 *>(src);
                        else w[k][0] = *reinterpret_cast<const uint32_t *>(src);
                    }
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        const uint8_t * src = vs + kv4_scale(D, 16 * j + 8 * k + 2 * c, 0);
                        if constexpr (NB == 4) *reinterpret_cast<uint4 *>(d[k]) = *reinterpret_cast<const uint4 *>(src);
                        else *reinterpret_cast<uint2 *>(d[k]) = *reinterpret_cast<const uint2 *>(src);
                        if (!whole) {   // a weight of zero does not silence a scale that is no number: cells nobody sees may hold anything
                            uint32_t keep2 = 0;
#pragma unroll
                            for (int e = 0; e < 2; e++) {
                                const int cell = base + 16 * j + 8 * k + 2 * c + e;
                                if (cell <= p_hi && (A.window <= 0 || p_lo - cell < A.window || cell < A.first)) keep2 |= 0xffffu << (16 * e);
                            }
#pragma unroll
                            for (int b = 0; b < NB; b++) d[k][b] &= keep2;
                        }
                    }
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        uint32_t v[2][4];   // [eight][number]: f16 of the two cells
#pragma unroll
                        for (int k = 0; k < 2; k++) {
                            const uint32_t u = __byte_perm(w[2 * k][b / 2], w[2 * k + 1][b / 2], b & 1 ? 0x7632 : 0x5410);
                            const __half2 sd = u2h(d[k][b]), s24 = __hmul2(sd, __float2half2_rn(-24.f));
                            v[k][0] = h2u(__hmul2(__hsub2(u2h((u & 0x000f000fu) | 0x64006400u), __float2half2_rn(1032.f)), sd));                // 1024 + n
                            v[k][1] = h2u(__hmul2(__hsub2(u2h((u & 0x00f000f0u) | 0x54005400u), __float2half2_rn(72.f)), sd));                  // 64 + n
                            v[k][2] = h2u(__hfma2(u2h((u >> 2 & 0x03c003c0u) | 0x4c004c00u), sd, s24));                                         // 16 + n: 24 scales are an f16
                            v[k][3] = h2u(__hfma2(u2h((u >> 6 & 0x03c003c0u) | 0x4c004c00u), sd, s24));
                        }
#pragma unroll
                        for (int h = 0; h < LO; h++) {
                            mma16816(o[b][0], v[0][0], v[0][1], v[1][0], v[1][1], pf[h][2 * j], pf[h][2 * j + 1]);
                            mma16816(o[b][1], v[0][2], v[0][3], v[1][2], v[1][3], pf[h][2 * j], pf[h][2 * j + 1]);
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
                if (g == 0) { part->m[r] = m[k]; part->l[r] = l[k]; }
            }
        }
        if (lane == 0) S.part[warp] = any ? part : nullptr;
        __syncthreads();
        const bool full = pa == 0 && pb == q.pages;
        KrPart<D> * ws = reinterpret_cast<KrPart<D> *>(W.parts);
        KrPart<D> * to = &ws[2 * blockIdx.x + (pa > 0 ? 0 : 1)];
        const int r = tid / (D / 4), d4 = 4 * (tid % (D / 4));
        auto joined = [&](auto && at, int n) {   // sum of n parts, in their order: (numbers, maximum, sum of weights)
            float top = -INFINITY, sum = 0.f;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int i = 0; i < n; i++)
                if (const KrPart<D> * p = at(i)) top = fmaxf(top, __ldcg(&p->m[r]));
            for (int i = 0; i < n; i++)
                if (const KrPart<D> * p = at(i)) {
                    const float mi = __ldcg(&p->m[r]), li = __ldcg(&p->l[r]);
                    const float f = mi == -INFINITY ? (li == li ? 0.f : 1.f) : ex2(mi - top);
                    const float4 y = __ldcg(reinterpret_cast<const float4 *>(&p->o[r][d4]));
                    sum += li * f;
                    x.x += y.x * f; x.y += y.y * f; x.z += y.z * f; x.w += y.w * f;
                }
            struct R { float4 x; float m, l; };
            return R{x, top, sum};
        };
        auto write = [&](float4 x, float sum) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            if (r < rows) store4(row_of(r) + d4, make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
        };
        if (r < KR_ROWS) {
            float top = -INFINITY, sum = 0.f;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
            for (int i = 0; i < KR_WARPS; i++)
                if (const KrPart<D> * p = S.part[i]) top = fmaxf(top, p->m[r]);
#pragma unroll 1
            for (int i = 0; i < KR_WARPS; i++)
                if (const KrPart<D> * p = S.part[i]) {
                    const float mi = p->m[r], li = p->l[r];
                    const float f = mi == -INFINITY ? (li == li ? 0.f : 1.f) : ex2(mi - top);
                    const float4 y = *reinterpret_cast<const float4 *>(&p->o[r][d4]);
                    sum += li * f;
                    x.x += y.x * f; x.y += y.y * f; x.z += y.z * f; x.w += y.w * f;
                }
            if (full) write(x, sum);
            else {
                *reinterpret_cast<float4 *>(&to->o[r][d4]) = x;
                if (d4 == 0) { to->m[r] = top; to->l[r] = sum; }
            }
        }
        if (!full) {
            const long long a0 = put.before + (long long) (tile * A.cache.n_head_kv + hk) * q.pages;   // the item's first unit
            const int c0 = (int) (a0 / share), c1 = (int) ((a0 + q.pages - 1) / share);                  // the CTAs that share it
            __threadfence();
            __syncthreads();
            if (tid == 0) S.last = atomicAdd(&W.counters[c0], 1) == c1 - c0;
            __syncthreads();
            if (S.last) {
                __threadfence();
                if (r < KR_ROWS) {
                    const auto j = joined([&](int i) { return &ws[2 * (c0 + i) + (i == 0 ? 1 : 0)]; }, c1 - c0 + 1);
                    write(j.x, j.l);
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
