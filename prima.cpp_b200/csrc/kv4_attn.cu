// prima.cpp_b200/csrc/kv4_attn.cu — attention over the 4-bit cache (kv4.cuh): which kernel takes a sequence.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>

#include "../../include/prima_b200.h"
#include "kv4_attn.cuh"

namespace pb {

// counters (rows: one per warp and slice), tickets and a word for each slot, all zero between calls; then the parts of either kernel, which may run at the same time
constexpr int KV4_SYNC = KV4_COUNTERS + 64 + KV4_SLOTS;      // and the words of calls with prefixes, which keep their place whatever a call's sizes
static size_t counters() { return (KV4_SYNC + 64) * sizeof(int); }
size_t kv4_attn_workspace(int D) { return counters() + kv4_rows_workspace(D) + kv4_prompt_workspace(D); }

static int few_rows(int type) { return type == PB200_TYPE_F32 ? KV4_FEW_ROWS_F32 : KV4_FEW_ROWS; }

int launch_kv4_attn(const Kv4Attn & a, int D, int type, void * ws, cudaStream_t st, int & launches) {
    int * words = (int *) ws;
    void * parts = (char *) ws + counters();
    const int64_t most = std::min<int64_t>(a.max_q, a.n_tokens) * a.group;
    const int few = few_rows(type);
    const bool ext = a.x.lse || a.x.mode != KV4_PLAIN;
    if (most <= few || a.n_seq > 1) {   // of several sequences, each goes where its rows belong
        launches++;
        const int e = launch_kv4_attn_rows(a, D, type, few, words, parts, st, ext);
        if (e || most <= few) return e;
    }
    // a single sequence is a prompt, as far as the host can tell: whatever rows it has
    return launch_kv4_attn_prompt(a, D, type, a.n_seq > 1 ? few : 0, words + KV4_COUNTERS, (char *) parts + kv4_rows_workspace(D), st, ext, launches);
}

// Rows' parts lie behind the workspace of a call without groups
static size_t round_up(size_t n) { return (n + 255) / 256 * 256; }
size_t kv4_attn_shared_workspace(int64_t rows, int D) { return round_up(kv4_attn_workspace(D)) + round_up((size_t) rows * D * sizeof(float)) + (size_t) rows * sizeof(float4); }

// A prefix is read once for the rows of all its sequences, by the prompts' kernel, where each sequence has few and these would walk many pages in front of their own; otherwise they do: nothing
// has to be added up, and there is one launch.  What counts is what is saved: pages (times kv heads and tiles of eight rows) that sequences would walk, less those that the prompts' kernel does, whose tile takes
// KV4_TILE times as long for a page whatever rows it has.  This is decided twice: the prompts' kernel is launched where tables have room for so many pages, all of one group's; it has
// work where there are half as many, as lengths, on the device: by then its launch, and the join's, have to be paid for anyway (8 us).
// us, pages in front of the own ones / by themselves, n sequences of one token in one group, 32 heads over 8, bf16: 1000 cells, 64 39 / 45, 128 55 / 46; 4000, 16 33 / 36, 24 41 / 40, 32 47 / 41, 128 123 / 63;
// 16 000, 8 46 / 49, 12 56 / 49, 32 117 / 51, 128 405 / 90; 16 heads over 2: 4000, 64 34 / 39, 128 47 / 46; F32, 32 over 8: 1000, 32 37 / 43, 64 56 / 46; 4000, 8 36 / 37, 12 39 / 38, 16 45 / 38;
// 16 000, 4 43 / 49, 8 67 / 54.  Groups of their own prefixes of 4000, bf16: 16 of 4 76 / 111, of 6 104 / 115, of 8 131 / 120, 4 of 12 66 / 55, 8 of 6 with a row each 67 / 73; F32: 16 of 3 99 / 141, of 4
// 119 / 144, of 6 168 / 149; 64 prefixes of one sequence each 75 / 339 (87 with the launch that has no work).  128 requests behind 16 009 cells, 5 to 900 of their own: 119 us, about 52 for the own cells, 55 for the prefix (0.4 of the tensor cores' rate) and 12 for the join
constexpr int KV4_APART = 8600, KV4_APART_F32 = 5000, KV4_TILE = 7, KV4_TILE_F32 = 5;
int launch_kv4_attn_shared(const Kv4Attn & a, const Kv4Groups & g, int D, int type, void * ws, cudaStream_t st, int & launches) {
    Kv4Attn b = a;
    int * words = (int *) ws;
    void * parts = (char *) ws + counters();
    b.x.sync = words + KV4_SYNC;
    b.x.o = (float *) ((char *) ws + round_up(kv4_attn_workspace(D)));
    b.x.ml = (float4 *) ((char *) b.x.o + round_up((size_t) a.n_tokens * a.n_head * D * sizeof(float)));
    b.x.group_start = g.start;
    b.x.prefix_len = g.kv_len;
    b.x.prefix_table = g.table;
    b.x.prefix_ld = g.table_ld;
    b.x.n_group = g.n;
    b.x.n_own = a.n_seq;
    b.x.room = (int) std::min<int64_t>(1 << 30, std::min<int64_t>(g.table_ld, 1 << 24) * KV4_CELLS);
    const bool f32 = type == PB200_TYPE_F32;
    const int few = few_rows(type);
    const int64_t most_q = std::min<int64_t>(a.max_q, a.n_tokens);
    int64_t least = 16 * (f32 ? KV4_APART_F32 : KV4_APART);
    b.x.mode = KV4_SHARED;
    // Sequences with few rows, and their tiles: those of the longest, but no more than all tokens make on the average; where there are sequences with many, these are taken for as few as have all
    // queries but one of each other, which are tokens; twice as much has to be saved there, since the prefix's kernel starts behind the prompts'.  us, pages in front of tokens' / by themselves, bf16, tokens and
    // a prompt of 512: behind 16 000 cells, 128 689 / 377, 28 272 / 246; 4000, 64 162 / 146, 28 114 / 124; one of 2000, 2000 cells, 64 190 / 213; F32, one of 200, 4000 cells, 64 207 / 168, 24 126 / 120
    int64_t n = a.n_seq, rows = most_q * a.group;
    double tiles = std::min<double>((rows + 7) / 8, 1 + (double) a.n_tokens * a.group / 8 / a.n_seq);
    if (rows > few) {
        b.x.few = few;
        least *= 2;
        n = a.group <= few && n > 1 ? n - (std::max<int64_t>(a.n_tokens - n, 0) + most_q - 2) / (most_q - 1) : 0;
        rows = std::min(a.group, few);
        tiles = (double) ((rows + 7) / 8);
    }
    b.x.of_seq = (int) (16 * a.cache.n_head_kv * tiles);
    b.x.of_tile = 16 * a.cache.n_head_kv * (f32 ? KV4_TILE_F32 : KV4_TILE);
    b.x.rows = (int) rows;
    b.x.log_tile = f32 ? 7 : 8;                  // rows of an item: kp_rows
    b.x.least = least / 2;
    const bool apart = n > 1 && (double) kv4_saved(b.x, n) * g.table_ld >= (double) least;
    if (!apart) b.x.least = INT64_MAX;
    const int e = launch_kv4_attn(b, D, type, ws, st, launches);
    if (e || !apart) return e;
    b.x.mode = KV4_FRONT;
    b.n_seq = g.n;
    return launch_kv4_attn_prompt(b, D, type, 0, words + KV4_COUNTERS, (char *) parts + kv4_rows_workspace(D), st, true, launches);
}

}  // namespace pb
