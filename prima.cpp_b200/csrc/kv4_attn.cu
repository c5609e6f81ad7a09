// prima.cpp_b200/csrc/kv4_attn.cu — attention over the 4-bit cache (kv4.cuh): which kernel takes a sequence.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "../../include/prima_b200.h"
#include "kv4_attn.cuh"

namespace pb {

// counters (rows: one per warp and slice), tickets and a word for each slot, all zero between calls; then the parts of either kernel, which may run at the same time
static size_t counters() { return (KV4_COUNTERS + 64 + KV4_SLOTS) * sizeof(int); }
size_t kv4_attn_workspace(int D) { return counters() + kv4_rows_workspace(D) + kv4_prompt_workspace(D); }

int launch_kv4_attn(const Kv4Attn & a, int D, int type, void * ws, cudaStream_t st, int & launches) {
    int * words = (int *) ws;
    void * parts = (char *) ws + counters();
    const int64_t most = std::min<int64_t>(a.max_q, a.n_tokens) * a.group;
    const int few = type == PB200_TYPE_F32 ? KV4_FEW_ROWS_F32 : KV4_FEW_ROWS;
    if (most <= few || a.n_seq > 1) {   // of several sequences, each goes where its rows belong
        launches++;
        const int e = launch_kv4_attn_rows(a, D, type, few, words, parts, st);
        if (e || most <= few) return e;
    }
    // a single sequence is a prompt, as far as the host can tell: whatever rows it has
    return launch_kv4_attn_prompt(a, D, type, a.n_seq > 1 ? few : 0, words + KV4_COUNTERS, (char *) parts + kv4_rows_workspace(D), st, launches);
}

}  // namespace pb
