// prima.cpp_b200/csrc/kv4_rows.cu — attention over the 4-bit cache (kv4.cuh) for sequences with few query rows: single tokens, drafts.
//
// Mathematics.  A sequence's queries that share a kv head are rows, token by token, the heads of the group next to each other; a tile has eight.  Products run on the
// tensor cores (m16n8k16, a row to a column: 16 cells or 16 numbers of a value x 8 rows), their 4-bit operand as it lies in the register: masked, n is the f16 n * 2^-24, or n * 2^-20 one
// nibble further up, exactly.
//   scores    with d a block's scale: q . k = sum over blocks b of d_b (sum_i q_i n_i - 8 sum_i q_i).  The sum over i is the product, which starts from what the 8 adds; scales go
//             onto the block's sums in 32 bits.  Numbers of the upper nibble meet queries of a 16th.
//   values    sum over cells of w d_b (n - 8): weights become the other operand transposed (movmatrix).  BF16: times the scales of their cells, the sum of which times 8 is a product with
//             constants; the power of two by which weights are larger than 2^(score - reference) follows the largest scale seen, so that neither they nor small products leave f16.  That rounds a
//             weight twice, an eighth of BF16's own rounding each.  F16 and F32: the 4-bit operand is made signed and scaled, exactly, and a weight is rounded once.  us, carried by the weights / by
//             the values: bf16, 32 sequences 52 / 53, two long ones 57.6 / 62, 40 of 8192 cells over 8 heads 82 / 91; f16, 256 of 1000 to 3000 132 / 145, and errors 3.05e-4 / 2.6e-4 (elementary
//             32-bit operations 2.1e-4, the output's rounding).
// With F32, queries and weights are two f16 numbers each (22 bits), and keys are made signed, too: products of n as it is, up to 15, lose 3e-6 to
// the tensor core's alignment of its 16 terms.  16-bit queries are one f16 number, exactly: a row is scaled by a power of two.
// Softmax by running maximum and sum, per page of 64 cells.
//
// Work.  The pages that a (sequence, tile, kv head) sees, all of them in a row, are dealt out to the warps in equal shares, so that lengths do not matter.  A warp walks its
// share by itself, pages on their way through a ring of its own (one bulk copy per page: a head's chunk is contiguous), and writes items that it has whole.  Of one that is cut it leaves
// its part in the workspace; once a CTA's warps are through, those that share an item add up its parts, and where it reaches beyond the CTA, the last warp of all adds
// what the CTAs have: always in their order (no atomics on numbers, equal calls give equal bits).  One barrier a CTA: with one per item, warps waited for each other for a
// page's time at every item (83 us for 32 sequences of up to 8192 cells; this 53).
//
// Bound: where there is much to read, half of the time is the memory's and half the start and the joins: of 57 us for two sequences of 131071 and 65001 cells (226 MB, 34.5 at the rate of a
// copy) 2 are the shares, 4 the wait for queries and first pages, 40 the pages (5300 clocks each for 12 warps of an SM, 19 bytes a clock and SM; with the values left out 5000: the copies
// set the pace), 6 the joins.  Where there is little, the chain of launch, lengths, page numbers, page, join: 14 us for a token behind 1000 cells.
// us: 32 sequences of 17 .. 8192 cells, 32 heads over 8, 53 (floor 24); 256 of 1000 .. 3000 132 (91); 16 in windows of 1024, heads of 64, 14.  Products on scaled values, a CTA's warps joining
// at every item, parts loaded one by one: 107, 79 and 22 for the first, the long two and the windows.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cfloat>
#include <type_traits>

#include "../../include/prima_b200.h"
#include "kv4_attn.cuh"

namespace pb {
namespace {

constexpr int KR_ROWS = 8;
// Warps of a CTA, one CTA to an SM: 168 registers (16 warps of 128: 94 us where these took 65, 8 warps of 234 the same).  Stages of a warp's ring: a page each.
constexpr int KR_WARPS = 12, KR_THREADS = 32 * KR_WARPS;
// Few pages go to as many warps of a CTA at least: one for each of an SM's schedulers.  us, with 4 / 8 / 12: a token of 32 heads over 8 behind 100 cells 11.6 / 15.4 / 19.1, behind
// 1000 13.6 / 15.2 / 20.1, behind 4000 17.1 / 17.9 / 19.5
constexpr int KR_LEAST = 4;
template <int D> constexpr int kr_stages() { return D == 128 ? 2 : 4; }
// Weights are 2^15 times 2^(score - reference), the largest 2^15 (F32: above 2^14): those of 2^-28 of it are normal f16 numbers, and what rounds off below them is 2^-40 (F32: of low parts, 2^-39)
constexpr int KR_UP = 15;

// a part of an item: sums of 2^(score - m) v, and of the weights
template <int D> struct KrPart { float o[KR_ROWS][D]; float m[KR_ROWS], l[KR_ROWS]; };
// workspace: parts of the warps (0: of an item that began before the warp's share, 1: of one that begins in it and goes on), parts of the CTAs in the same way
template <int D> struct KrParts { KrPart<D> warp[KV4_MAX_CTAS * KR_WARPS][2], cta[KV4_MAX_CTAS][2]; };

// A segment: pages [pa, pb) (of those that it sees) of an item, which are the units k0 .. u - 1.
struct KrSegment {
    Kv4Seq q;
    int s, before;             // the sequence, units in front of it
    int u;                     // the unit behind the segment
    int tile, hk, pa, pb, k0;
};
template <int D> struct __align__(128) KrSmem {
    __align__(128) uint8_t ring[KR_WARPS][kr_stages<D>()][kv4_chunk_bytes(D)];
    uint64_t full[KR_WARPS][kr_stages<D>()];
    KrSegment get[KR_WARPS];   // where each warp's fetching is
    KrSegment begin[KR_WARPS];
    KrSegment cut[KR_WARPS][2];       // items of which a warp has a part: one that began before its share, one that goes on
    const KrPart<D> * part[KR_WARPS][2];
    int scan[KR_WARPS];
    int abort;
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
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
template <typename T> __device__ __forceinline__ float2 to_f32x2(uint32_t w) {
    if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2 *>(&w));
    else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ uint32_t h2u(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
__device__ __forceinline__ __half2 u2h(uint32_t u) { return *reinterpret_cast<__half2 *>(&u); }

// four numbers of a row of an item: parts added up in their order
struct KrSum {
    float top = -INFINITY, l = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    // ONCE parts on their way together; far: of other CTAs, from L2
    template <int ONCE, bool FAR, typename At>
    __device__ __forceinline__ void add(int n, int r, int d4, At && at) {
        for (int i0 = 0; i0 < n; i0 += ONCE) {
            float mi[ONCE], li[ONCE], t = top;
            float4 y[ONCE];
#pragma unroll
            for (int k = 0; k < ONCE; k++) {
                const auto * p = at(min(i0 + k, n - 1));
                const float4 * o = reinterpret_cast<const float4 *>(&p->o[r][d4]);
                mi[k] = FAR ? __ldcg(&p->m[r]) : p->m[r];
                li[k] = FAR ? __ldcg(&p->l[r]) : p->l[r];
                y[k] = FAR ? __ldcg(o) : *o;
            }
#pragma unroll
            for (int k = 0; k < ONCE; k++) t = fmaxf(t, mi[k]);
            const float f = part_factor(top, l, t);
            top = t;
            l *= f;
            x.x *= f; x.y *= f; x.z *= f; x.w *= f;
#pragma unroll
            for (int k = 0; k < ONCE; k++)
                if (i0 + k < n) {
                    const float h = part_factor(mi[k], li[k], t);
                    l = fmaf(li[k], h, l);
                    x.x = fmaf(y[k].x, h, x.x); x.y = fmaf(y[k].y, h, x.y); x.z = fmaf(y[k].z, h, x.z); x.w = fmaf(y[k].w, h, x.w);
                }
        }
    }
    template <typename T> __device__ __forceinline__ void write(T * to) const {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        store4(to, make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
    }
    template <typename T> __device__ __forceinline__ void write(T * to, const Kv4Row & r, int d4) const {
        if (r.put) store4(r.put + d4, x);
        else store4(to, kv4_mix(r, x, d4));
    }
};
// row r of a segment's tile in the output
template <typename T, int D>
__device__ __forceinline__ T * kr_row(const Kv4Attn & A, const KrSegment & at, int r) {
    const int row = at.tile * KR_ROWS + r, t = row / A.group;
    return (T *) A.out + (at.q.q0 + t) * A.ldo + (int64_t) (at.hk * A.group + row - t * A.group) * D;
}
template <int D>
__device__ __forceinline__ Kv4Row kr_ext(const Kv4Attn & A, const KrSegment & at, int r, float m, float l, bool writes) {
    const int row = at.tile * KR_ROWS + r, t = row / A.group;
    return kv4_row<D>(A, at.q, at.q.q0 + t, at.hk * A.group + row - t * A.group, m, l, writes);
}

template <typename T, int D, bool X>
__global__ void __launch_bounds__(KR_THREADS, 1) k_kv4_attn_rows(const __grid_constant__ Kv4Attn A, const __grid_constant__ KrWork W) {
    constexpr int NB = D / 32, STAGES = kr_stages<D>(), CHUNK = kv4_chunk_bytes(D);
    constexpr bool F32 = std::is_same<T, float>::value, SCALED = std::is_same<T, __nv_bfloat16>::value;   // SCALED: weights carry the values' scales
    constexpr int LO = F32 ? 2 : 1;
    extern __shared__ uint8_t smem_raw[];
    KrSmem<D> & S = *reinterpret_cast<KrSmem<D> *>(smem_raw + ((128u - (smem_u32(smem_raw) & 127u)) & 127u));
    const int tid = threadIdx.x, warp = uniform_warp(), lane = tid & 31, g = lane >> 2, c = lane & 3;
    volatile int * cta_abort = &S.abort;
    const int hks = A.cache.n_head_kv;

    pdl_trigger();                                      // the prompts' kernel may start where this one has no work

    // ---- shares: units (pages of items) in the order of sequences, tiles, heads, pages; a thread has a sequence ----
    Kv4Seq mine = kv4_seq<X>(A, tid, W.most_rows, false);
    int n = mine.units(hks, KR_ROWS), units = n;
    if (lane < STAGES) {
        mbar_init(&S.full[warp][lane], 1);
        mbar_fence_init();
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (tid == 0) S.abort = 0;
    for (int s = tid + KR_THREADS; s < A.n_seq; s += KR_THREADS) units += kv4_seq<X>(A, s, W.most_rows, false).units(hks, KR_ROWS);
    auto upto = [&](int x) {                   // sum over the lanes up to this one
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        return x;
    };
    int x = upto(units);
    if (lane == 31) S.scan[warp] = x;
    __syncthreads();
    int total = 0, front = 0;
#pragma unroll
    for (int w = 0; w < KR_WARPS; w++) {
        const int k = S.scan[w];
        if (w < warp) front += k;
        total += k;
    }
    if (total == 0) return;
    // warps at work in a CTA: few pages go to one warp of each of an SM's four schedulers, on as many SMs as that takes
    const int at_work = total >= (int) gridDim.x * KR_WARPS ? KR_WARPS : max(KR_LEAST, (total + (int) gridDim.x - 1) / (int) gridDim.x);
    const int share = (int) (((unsigned) total + gridDim.x * at_work - 1) / (gridDim.x * at_work));
    const int me = blockIdx.x * at_work + warp;
    // the sequences in which the warps' shares begin
    const long long cta0 = (long long) blockIdx.x * at_work * share;
    auto begins = [&](const Kv4Seq & q, int s, int before, int n) {
        if (before >= cta0 + (long long) at_work * share || before + n <= cta0) return;
#pragma unroll 1
        for (int w = 0; w < at_work; w++) {
            const long long u = cta0 + w * share;
            if (u >= before && u < before + n) {
                S.begin[w].q = q;
                S.begin[w].s = s;
                S.begin[w].before = before;
            }
        }
    };
    if (A.n_seq <= KR_THREADS) begins(mine, tid, front + x - n, n);
    else {
        int before = 0;
        for (int s0 = 0; s0 < A.n_seq; s0 += KR_THREADS) {
            mine = kv4_seq<X>(A, s0 + tid, W.most_rows, false);
            n = mine.units(hks, KR_ROWS);
            x = upto(n);
            __syncthreads();
            if (lane == 31) S.scan[warp] = x;
            __syncthreads();
            front = before;
            for (int w = 0; w < KR_WARPS; w++) {
                if (w < warp) front += S.scan[w];
                before += S.scan[w];
            }
            begins(mine, s0 + tid, front + x - n, n);
        }
    }
    __syncthreads();
    const long long u0_ = cta0 + (long long) warp * share;
    const int u0 = warp < at_work && u0_ < total ? (int) u0_ : total, u1 = total - u0 < share ? total : u0 + share;

    // the segment that begins at p.u: false if there is none in the share
    auto next = [&](KrSegment & p) {
        if (p.u >= u1) return false;
        while (p.u - p.before >= p.q.units(hks, KR_ROWS)) {
            p.before += p.q.units(hks, KR_ROWS);
            if (++p.s >= A.n_seq) return false;
            p.q = kv4_seq<X>(A, p.s, W.most_rows, false);
        }
        const int in = p.u - p.before, item = in / p.q.pages;
        p.pa = in - item * p.q.pages;
        p.pb = min(p.q.pages, p.pa + u1 - p.u);
        p.tile = item / hks;
        p.hk = item - p.tile * hks;
        p.k0 = p.u;
        p.u += p.pb - p.pa;
        return true;
    };
    KrSegment put;
    bool more = false;
    if (u0 < u1) {
        put = S.begin[warp];
        put.u = u0;
        more = next(put);
    }
    // queries of a segment: lane (g, c) has of row g the numbers 32 b + 8 c + e
    constexpr int RAW = F32 ? 4 : 2;
    uint32_t raw[NB][2][RAW];
    auto ask = [&](const KrSegment & p) {
        const int row = p.tile * KR_ROWS + g;
        const bool have = row < p.q.n_rows;
        const int t = row / A.group;
        const T * src = (const T *) A.q + (p.q.q0 + t) * A.ldq + (int64_t) (p.hk * A.group + row - t * A.group) * D + 8 * c;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                if constexpr (F32) {
                    const uint4 w = have ? *reinterpret_cast<const uint4 *>(src + 32 * b + 4 * h) : make_uint4(0u, 0u, 0u, 0u);
                    raw[b][h][0] = w.x; raw[b][h][1] = w.y; raw[b][h][2] = w.z; raw[b][h][3] = w.w;
                } else {
                    const uint2 w = have ? *reinterpret_cast<const uint2 *>(src + 32 * b + 4 * h) : make_uint2(0u, 0u);
                    raw[b][h][0] = w.x; raw[b][h][1] = w.y;
                }
            }
    };
    if (more) ask(put);                                 // ahead of the pages, which fill the memory's queues

    // ---- pages on their way: unit u goes through stage (u - u0) % STAGES ----
    uint64_t policy;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    if (more && lane == 0) S.get[warp] = put;
    __syncwarp();
    uint32_t none = 0;                                  // stages whose page is none: nothing is on its way
    int ids = -1, ids0 = 0, ids1 = 0, f_hk = 0;         // page numbers of the units ids0 .. ids1 - 1 of a segment, one to a lane; its kv head
    auto fetch = [&](int u) {                           // by ascending u
        if (u >= u1) return;
        if (u >= ids1) {
            KrSegment p = S.get[warp];
            if (u >= p.u) {
                next(p);
                __syncwarp();
                if (lane == 0) S.get[warp] = p;
                __syncwarp();
            }
            ids0 = u;
            ids1 = min(u + 32, p.u);
            f_hk = p.hk;
            ids = u + lane < ids1 ? kv4_page<X>(A, p.q, p.s, p.pa + u + lane - p.k0) : -1;
        }
        const int id = __shfl_sync(0xffffffffu, ids, u - ids0), st = (u - u0) % STAGES;
        none = id >= 0 ? none & ~(1u << st) : none | 1u << st;
        if (elect_one()) {
            if (id >= 0) {
                mbar_arrive_expect_tx(&S.full[warp][st], CHUNK);
                bulk_g2s(S.ring[warp][st], kv4_chunk<D>(A.cache, id, f_hk), CHUNK, &S.full[warp][st], policy);
            } else mbar_arrive(&S.full[warp][st]);
        }
        __syncwarp();
    };
    // ---- segments ----
    KrParts<D> & parts = *reinterpret_cast<KrParts<D> *>(W.parts);
    if (lane < 2) S.cut[warp][lane].q.n_q = 0;
    __syncwarp();
    while (more) {
        const KrSegment at = put;
        const Kv4Seq & q = at.q;
        const int row0 = at.tile * KR_ROWS, rows = min(KR_ROWS, q.n_rows - row0);
        // queries as pairs; F32: two f16 numbers each (high, low), otherwise pairs 1 and 3 a 16th
        uint32_t qf[LO][NB][4];
        float start[NB][2], mult[2];
        int pos[2];
        {
            float x[NB][8], top = 0.f;
            const int row = row0 + g;
            const bool have = g < rows;
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    if constexpr (F32) {
#pragma unroll
                        for (int e = 0; e < 4; e++) x[b][4 * h + e] = __uint_as_float(raw[b][h][e]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const float2 v = to_f32x2<T>(raw[b][h][e]);
                            x[b][4 * h + 2 * e] = v.x;
                            x[b][4 * h + 2 * e + 1] = v.y;
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 4; e++) top = fmaxf(top, fabsf(x[b][4 * h + e]));
                }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // the row's power of two: its largest number comes to 2^13 .. 2^14
            const int ex = top > 0.f && top < INFINITY ? min(126, 140 - (int) (__float_as_uint(top) >> 23)) : 0;
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
            const int p = kv4_pos<X>(A, q, row / A.group);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int from = 4 * (2 * c + i);                               // a lane of row 2 c + i
                mult[i] = __shfl_sync(0xffffffffu, down, from);
                pos[i] = __shfl_sync(0xffffffffu, have ? p : -1, from);
#pragma unroll
                for (int b = 0; b < NB; b++) start[b][i] = F32 ? 0.f : __shfl_sync(0xffffffffu, sums[b], from);
            }
        }
        if (at.k0 == u0)                                // the first pages, behind the queries: these would wait for all that is on its way to this SM
            for (int k = 0; k < STAGES; k++) fetch(u0 + k);
        const int2 hole = kv4_hole<X>(A, q);
        const int p_lo = kv4_pos<X>(A, q, row0 / A.group), p_hi = kv4_pos<X>(A, q, (row0 + rows - 1) / A.group);   // of the tile's rows

        // out^T: lane: numbers 32 b + 4 g + 2 h, + 1 of rows 2 c, 2 c + 1 (SCALED: times 2^-24, and 2^-20 the odd ones)
        float o[NB][2][4], less[4] = {0.f, 0.f, 0.f, 0.f};     // less: SCALED: row b: - 8 * 2^-24 times the sum of block b's scaled weights
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
        int up = KR_UP;                                 // weights are 2^(score - reference + up)
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 4; i++) o[b][0][i] = o[b][1][i] = 0.f;
        for (int u = at.k0; u < at.u; u++) {
            const int st = (u - u0) % STAGES;
            const bool have = !(none >> st & 1);
            mbar_wait(&S.full[warp][st], (uint32_t) ((u - u0) / STAGES) & 1, cta_abort, W.abort_flag);
            if (have) {
                uint8_t * chunk = S.ring[warp][st];
                uint8_t * const vs = chunk + 2 * kv4_rows_bytes(D) + kv4_scales_bytes(D);
                const int base = kv4_page_index<X>(A, q, at.pa + u - at.k0) * KV4_CELLS;
                const bool whole = base + 63 <= p_lo && (A.window <= 0 || p_hi - base < A.window || base + 63 < A.first) && !kv4_has_hole<X>(hole, base);
                if (!whole) {   // a weight of zero does not silence a scale that is no number: cells nobody sees may hold anything
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int t = 2 * lane + e, cell = base + t;
                        if (!(cell <= p_hi && (A.window <= 0 || p_lo - cell < A.window || cell < A.first)) || kv4_in_hole<X>(hole, cell))
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
                    for (int b = 0; b < NB; b++) {
                        float acc[4];
                        const uint32_t a1 = wa[b] >> 8, b1 = wb[b] >> 8;
                        if constexpr (F32) {
                            auto even = [](uint32_t w) { return h2u(__hsub2(u2h((w & 0x000f000fu) | 0x64006400u), __float2half2_rn(1032.f))); };   // 1024 + n
                            auto odd = [](uint32_t w) { return h2u(__hsub2(u2h((w & 0x00f000f0u) | 0x54005400u), __float2half2_rn(72.f))); };      // 64 + n
                            const uint32_t x[8] = {even(wa[b]), even(wb[b]), odd(wa[b]), odd(wb[b]), even(a1), even(b1), odd(a1), odd(b1)};      // low parts of the queries first
                            mma16816_from(acc, 0.f, 0.f, x[0], x[1], x[2], x[3], qf[LO - 1][b][0], qf[LO - 1][b][1]);
                            mma16816(acc, x[4], x[5], x[6], x[7], qf[LO - 1][b][2], qf[LO - 1][b][3]);
                            mma16816(acc, x[0], x[1], x[2], x[3], qf[0][b][0], qf[0][b][1]);
                            mma16816(acc, x[4], x[5], x[6], x[7], qf[0][b][2], qf[0][b][3]);
                        } else {
                            mma16816_from(acc, start[b][0], start[b][1], wa[b] & 0x000f000fu, wb[b] & 0x000f000fu, wa[b] & 0x00f000f0u, wb[b] & 0x00f000f0u, qf[0][b][0], qf[0][b][1]);
                            mma16816(acc, a1 & 0x000f000fu, b1 & 0x000f000fu, a1 & 0x00f000f0u, b1 & 0x00f000f0u, qf[0][b][2], qf[0][b][3]);
                        }
                        const float da = __half2float(*reinterpret_cast<const __half *>(ks + 4 * b)), db = __half2float(*reinterpret_cast<const __half *>(ks + 4 * b + 16 * NB));
                        sc[j][0] = b == 0 ? acc[0] * da : fmaf(acc[0], da, sc[j][0]);
                        sc[j][1] = b == 0 ? acc[1] * da : fmaf(acc[1], da, sc[j][1]);
                        sc[j][2] = b == 0 ? acc[2] * db : fmaf(acc[2], db, sc[j][2]);
                        sc[j][3] = b == 0 ? acc[3] * db : fmaf(acc[3], db, sc[j][3]);
                    }
                }
                if (!whole) {
#pragma unroll
                    for (int j = 0; j < 4; j++)
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const int cell = base + 16 * j + g + (k >> 1) * 8, p = pos[k & 1];
                            if (!(cell <= p && (A.window <= 0 || p - cell < A.window || cell < A.first)) || kv4_in_hole<X>(hole, cell)) sc[j][k] = -INFINITY;
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
                    // rounded upwards, so that weights stay within 2^up however large scores are.  F32: to a whole number: what weights, sums and parts are scaled by are powers of two then
                    // (16 bits: the largest weight is a power of two, which f16 holds exactly; rounded, errors are a third larger)
                    mx[k] = __fmul_ru(a, mult[k]);
                    if constexpr (F32) mx[k] = ceilf(mx[k]);
                }
                int to = up;
                if constexpr (SCALED) {   // lane: the scales of cells 2 lane, 2 lane + 1
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
                        if (SCALED && b == 0) {
                            less[0] *= f[0]; less[1] *= f[1];
                        }
                    }
                }
                const float off[2] = {m[0] == -INFINITY ? 0.f : __fsub_rd((float) up, m[0]), m[1] == -INFINITY ? 0.f : __fsub_rd((float) up, m[1])};
                // weights, transposed: lane: row g, cells 8 x + 2 c, + 1 (x: eights of the page)
                uint32_t pf[LO][8];
#pragma unroll
                for (int x8 = 0; x8 < 8; x8++) {
                    const float e0 = ex2(fmaf(sc[x8 >> 1][2 * (x8 & 1)], mult[0], off[0])), e1 = ex2(fmaf(sc[x8 >> 1][2 * (x8 & 1) + 1], mult[1], off[1]));
                    l[0] += e0;
                    l[1] += e1;
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
                        if constexpr (!SCALED) {
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
                            for (int h = 0; h < 2; h++) {
                                if constexpr (F32) {
                                    // 16 cells' products start from zero, low parts of the weights first, and are added to the sums in 32 bits: the tensor core cuts off what it adds to, and a sum
                                    // that ran through all cells lost with their number (40 sequences of 8192 cells 3.9e-6)
                                    float t[4];
                                    mma16816_from(t, 0.f, 0.f, v[0][2 * h], v[0][2 * h + 1], v[1][2 * h], v[1][2 * h + 1], pf[LO - 1][2 * j], pf[LO - 1][2 * j + 1]);
                                    mma16816(t, v[0][2 * h], v[0][2 * h + 1], v[1][2 * h], v[1][2 * h + 1], pf[0][2 * j], pf[0][2 * j + 1]);
#pragma unroll
                                    for (int i = 0; i < 4; i++) o[b][h][i] += t[i];
                                } else mma16816(o[b][h], v[0][2 * h], v[0][2 * h + 1], v[1][2 * h], v[1][2 * h + 1], pf[0][2 * j], pf[0][2 * j + 1]);
                            }
                        } else {
                            const uint32_t p0 = h2u(__hmul2(u2h(pf[0][2 * j]), u2h(d[0][b]))), p1 = h2u(__hmul2(u2h(pf[0][2 * j + 1]), u2h(d[1][b])));
                            const uint32_t s0 = u[0] >> 8, s1 = u[1] >> 8;
                            mma16816(o[b][0], u[0] & 0x000f000fu, u[0] & 0x00f000f0u, u[1] & 0x000f000fu, u[1] & 0x00f000f0u, p0, p1);
                            mma16816(o[b][1], s0 & 0x000f000fu, s0 & 0x00f000f0u, s1 & 0x000f000fu, s1 & 0x00f000f0u, p0, p1);
                            const uint32_t eights = g == b ? 0x80088008u : 0u;
                            mma16816(less, eights, 0u, eights, 0u, p0, p1);
                        }
                    }
                }
            }
            __syncwarp();
            fetch(u + STAGES);
        }
        more = next(put);
        if (more) ask(put);                             // the next item's queries, on their way meanwhile
#pragma unroll
        for (int k = 0; k < 2; k++) {
            l[k] += __shfl_xor_sync(0xffffffffu, l[k], 4);
            l[k] += __shfl_xor_sync(0xffffffffu, l[k], 8);
            l[k] += __shfl_xor_sync(0xffffffffu, l[k], 16);
        }
        if constexpr (SCALED)
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const float n8 = __shfl_sync(0xffffffffu, less[k], 4 * b + c);
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        o[b][h][k] = (o[b][h][k] + n8) * 16777216.f;
                        o[b][h][2 + k] = fmaf(n8, 16.f, o[b][h][2 + k]) * 1048576.f;
                    }
                }
        if (at.pa == 0 && at.pb == q.pages) {
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const int r = 2 * c + k;
                const float inv = l[k] == 0.f ? 0.f : 1.f / l[k];
                if (X && r < rows) {
                    const Kv4Row w = kr_ext<D>(A, at, r, m[k] - (float) up, l[k], g == 0);
                    T * to = kr_row<T, D>(A, at, r) + 4 * g;
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        const float4 x = make_float4(o[b][0][k], o[b][0][2 + k], o[b][1][k], o[b][1][2 + k]);
                        if (w.put) store4(w.put + 32 * b + 4 * g, x);
                        else store4(to + 32 * b, kv4_mix(w, x, 32 * b + 4 * g));
                    }
                } else if (r < rows) {
                    T * to = kr_row<T, D>(A, at, r) + 4 * g;
#pragma unroll
                    for (int b = 0; b < NB; b++) store4(to + 32 * b, make_float4(o[b][0][k] * inv, o[b][0][2 + k] * inv, o[b][1][k] * inv, o[b][1][2 + k] * inv));
                }
            }
        } else {
            // a part: where the share ends, through the warp's ring, which is empty then
            const int which = at.pa > 0 ? 0 : 1;
            KrPart<D> & to = more ? parts.warp[me][which] : *reinterpret_cast<KrPart<D> *>(S.ring[warp][0]);
            if (lane == 0) {
                S.cut[warp][which] = at;
                S.part[warp][which] = &to;
            }
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const int r = 2 * c + k;
#pragma unroll
                for (int b = 0; b < NB; b++) *reinterpret_cast<float4 *>(&to.o[r][32 * b + 4 * g]) = make_float4(o[b][0][k], o[b][0][2 + k], o[b][1][k], o[b][1][2 + k]);
                if (g == 0) { to.m[r] = m[k] - (float) up; to.l[r] = l[k]; }
            }
        }
    }

    // ---- items that were cut ----
    __syncthreads();                                    // the CTA's parts are there
    // of each, slices of 32 x 4 numbers, which go to the CTA's warps in turns; where the item reaches beyond the CTA, the last of the CTAs to come adds theirs
    constexpr int SLICES = KR_ROWS * D / 128;
    static_assert(SLICES <= KR_WARPS && 2 * KR_WARPS <= 32, "a warp has a slice of an item at most, a lane of it an item");
    const int first = blockIdx.x * at_work;
    int w0 = 0, w1 = 0, f1 = 0;                          // lane: the warps that share item `lane`, the last of them in this CTA
    bool here = false;                                   // (each item once: where its first warp in this CTA stands)
    if (lane < 2 * at_work && S.cut[lane >> 1][lane & 1].q.n_q > 0) {
        const KrSegment & at = S.cut[lane >> 1][lane & 1];
        const int a0 = at.before + (at.tile * hks + at.hk) * at.q.pages;             // the item's first unit
        w0 = a0 / share;
        w1 = (a0 + at.q.pages - 1) / share;
        f1 = min(w1, first + at_work - 1);
        here = max(w0, first) == first + (lane >> 1);
    }
    uint32_t tasks = 0;                                  // items of which this warp has a slice that is to be joined with other CTAs'; lane: its counter
    int counter = 0, others = 0, turn = warp;
    auto item = [&](int k, auto && f) {                  // f(segment, slice, its warps)
        const int b = turn % KR_WARPS;
        if (b >= SLICES) return;
        const KrSegment & at = S.cut[k >> 1][k & 1];
        const int v0 = __shfl_sync(0xffffffffu, w0, k), v1 = __shfl_sync(0xffffffffu, w1, k), e = b * 32 + lane;
        f(at, b, v0, v1, e / (D / 4), 4 * (e % (D / 4)), min(KR_ROWS, at.q.n_rows - at.tile * KR_ROWS));
    };
    for (uint32_t left = __ballot_sync(0xffffffffu, here); left; left &= left - 1, turn += KR_WARPS - SLICES) {
        const int k = __ffs((int) left) - 1, to = __shfl_sync(0xffffffffu, f1, k);
        item(k, [&](const KrSegment & at, int b, int v0, int v1, int r, int d4, int rows) {
            const int f0 = max(v0, first);
            KrSum sum;
            sum.add<KR_WARPS, false>(to - f0 + 1, r, d4, [&](int i) { return S.part[f0 - first + i][f0 + i == v0 ? 1 : 0]; });
            if (v0 >= first && v1 < first + at_work) {
                if (r >= rows) return;
                if constexpr (X) sum.write(kr_row<T, D>(A, at, r) + d4, kr_ext<D>(A, at, r, sum.top, sum.l, d4 == 0), d4);
                else sum.write(kr_row<T, D>(A, at, r) + d4);
                return;
            }
            KrPart<D> & mid = parts.cta[blockIdx.x][f0 == v0 ? 1 : 0];
            *reinterpret_cast<float4 *>(&mid.o[r][d4]) = sum.x;
            if (d4 == 0) { mid.m[r] = sum.top; mid.l[r] = sum.l; }
            tasks |= 1u << k;
            if (lane == k) {
                counter = v0 * SLICES + b;
                others = v1 / at_work - v0 / at_work;
            }
        });
    }
    if (!tasks) return;
    __syncwarp();
    bool last = false;
    if (tasks >> lane & 1) {
        __threadfence();                                 // behind the warp's barrier: all its lanes' numbers
        last = atomicAdd(&W.counters[counter], 1) == others;
        if (last) W.counters[counter] = 0;
        __threadfence();
    }
    const uint32_t mine_last = __ballot_sync(0xffffffffu, last);
    turn = warp;
    for (uint32_t left = __ballot_sync(0xffffffffu, here); left; left &= left - 1, turn += KR_WARPS - SLICES) {
        const int k = __ffs((int) left) - 1;
        if (!(mine_last >> k & 1)) continue;
        item(k, [&](const KrSegment & at, int, int v0, int v1, int r, int d4, int rows) {
            const int c0 = v0 / at_work, c1 = v1 / at_work;
            KrSum sum;
            sum.add<16, true>(c1 - c0 + 1, r, d4, [&](int i) { return &parts.cta[c0 + i][i == 0 ? 1 : 0]; });
            if (r >= rows) return;
            if constexpr (X) sum.write(kr_row<T, D>(A, at, r) + d4, kr_ext<D>(A, at, r, sum.top, sum.l, d4 == 0), d4);
            else sum.write(kr_row<T, D>(A, at, r) + d4);
        });
    }
}

template <typename T, int D, bool X>
int rows_launch(const Kv4Attn & a, const KrWork & w, cudaStream_t st) {
    constexpr size_t smem = sizeof(KrSmem<D>) + 128;
    static_assert(smem <= 232448, "shared memory of an SM");
    static FuncAttrCache cache;
    const cudaError_t e = ensure_dyn_smem(cache, (const void *) k_kv4_attn_rows<T, D, X>, smem, true);
    if (e != cudaSuccess) return (int) e;
    k_kv4_attn_rows<T, D, X><<<sm_count() < KV4_MAX_CTAS ? sm_count() : KV4_MAX_CTAS, KR_THREADS, smem, st>>>(a, w);
    return (int) cudaGetLastError();
}

}  // namespace

size_t kv4_rows_workspace(int D) { return D == 128 ? sizeof(KrParts<128>) : sizeof(KrParts<64>); }
static_assert(sizeof(KrPart<128>) <= kv4_chunk_bytes(128) && sizeof(KrPart<64>) <= kv4_chunk_bytes(64), "a part goes through a stage");
static_assert(KV4_COUNTERS >= KV4_MAX_CTAS * KR_WARPS * KR_ROWS, "a counter for each slice of a warp's item");

template <int D, bool X>
static int rows_launch(const Kv4Attn & a, const KrWork & w, int type, cudaStream_t st) {
    return type == PB200_TYPE_F32 ? rows_launch<float, D, X>(a, w, st) : type == PB200_TYPE_F16 ? rows_launch<__half, D, X>(a, w, st) : rows_launch<__nv_bfloat16, D, X>(a, w, st);
}
int launch_kv4_attn_rows(const Kv4Attn & a, int D, int type, int most_rows, int * counters, void * parts, cudaStream_t st, bool ext) {
    const KrWork w{most_rows, counters, parts, abort_flag()};
    if (ext) return D == 128 ? rows_launch<128, true>(a, w, type, st) : rows_launch<64, true>(a, w, type, st);
    return D == 128 ? rows_launch<128, false>(a, w, type, st) : rows_launch<64, false>(a, w, type, st);
}

}  // namespace pb
