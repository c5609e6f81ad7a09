// prima.cpp_b200/csrc/kv4_attn.cu — attention over the 4-bit cache (kv4.cuh): which kernel takes a sequence.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>

#include "../../include/prima_b200.h"
#include "kv4_attn.cuh"

namespace pb {

// counters (rows: one per warp and slice), tickets and a word for each slot, all zero between calls; then the parts of either kernel, which may run at the same time
static size_t counters() { return (KV4_COUNTERS + 64 + KV4_SLOTS) * sizeof(int); }
size_t kv4_attn_workspace(int D) { return counters() + kv4_rows_workspace(D) + kv4_prompt_workspace(D); }

static int few_rows(int type) { return type == PB200_TYPE_F32 ? KV4_FEW_ROWS_F32 : KV4_FEW_ROWS; }

int launch_kv4_attn(const Kv4Attn & a, int D, int type, void * ws, cudaStream_t st, int & launches) {
    int * words = (int *) ws;
    void * parts = (char *) ws + counters();
    const int64_t most = std::min<int64_t>(a.max_q, a.n_tokens) * a.group;
    const int few = few_rows(type);
    const bool ext = a.x.lse || a.x.part;
    if (most <= few || a.n_seq > 1) {   // of several sequences, each goes where its rows belong
        launches++;
        const int e = launch_kv4_attn_rows(a, D, type, few, words, parts, st, ext);
        if (e || most <= few) return e;
    }
    // a single sequence is a prompt, as far as the host can tell: whatever rows it has
    return launch_kv4_attn_prompt(a, D, type, a.n_seq > 1 ? few : 0, words + KV4_COUNTERS, (char *) parts + kv4_rows_workspace(D), st, ext, launches);
}

// Rows' parts lie behind the workspace of a call without groups.
static size_t part_rows(int64_t rows, int D) { return ((size_t) rows * D * sizeof(float) + 255) / 256 * 256; }
size_t kv4_attn_shared_workspace(int64_t rows, int D) { return (kv4_attn_workspace(D) + 255) / 256 * 256 + part_rows(rows, D) + (size_t) rows * sizeof(float2); }

// The prefixes first: a group is a sequence whose rows all see all cells.  Which kernel takes them is decided for the call: by the rows that a group has on the average.
int launch_kv4_attn_shared(const Kv4Attn & a, const Kv4Groups & g, int D, int type, void * ws, cudaStream_t st, int & launches) {
    Kv4Attn own = a, front = a;
    own.x.o = front.x.o = (float *) ((char *) ws + (kv4_attn_workspace(D) + 255) / 256 * 256);
    own.x.ml = front.x.ml = (float2 *) ((char *) own.x.o + part_rows(a.n_tokens * a.n_head, D));
    own.x.group_start = front.x.group_start = g.start;
    own.x.n_group = front.x.n_group = g.n;
    own.x.n_seq = front.x.n_seq = a.n_seq;
    own.x.part = KV4_FOLD;
    front.x.part = KV4_PUT;
    front.x.all = 1;
    front.x.lse = nullptr;
    front.n_seq = g.n;
    front.kv_len = g.kv_len;
    front.table = g.table;
    front.table_ld = g.table_ld;
    front.max_q = INT_MAX;
    int * words = (int *) ws;
    void * parts = (char *) ws + counters();
    int e;
    if (a.n_tokens * a.group <= (int64_t) few_rows(type) * g.n) {
        launches++;
        e = launch_kv4_attn_rows(front, D, type, INT_MAX, words, parts, st, true);
    } else e = launch_kv4_attn_prompt(front, D, type, 0, words + KV4_COUNTERS, (char *) parts + kv4_rows_workspace(D), st, true, launches);
    return e ? e : launch_kv4_attn(own, D, type, ws, st, launches);
}

}  // namespace pb
