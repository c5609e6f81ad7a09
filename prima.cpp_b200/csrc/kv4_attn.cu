// prima.cpp_b200/csrc/kv4_attn.cu — attention over the 4-bit cache (kv4.cuh): which kernel takes a sequence.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "kv4_attn.cuh"

namespace pb {

// A sequence with up to so many rows (queries x heads of a group) goes to the kernel of few rows, which walks its pages once for every eight of them.
constexpr int KV4_FEW_ROWS = 16;

// counters (rows: one per warp and slice, zero between calls), tickets and a word for each slot, then the parts of either kernel, which run one after the other
static size_t counters() { return (KV4_COUNTERS + 64 + KV4_SLOTS) * sizeof(int); }
size_t kv4_attn_workspace(int D, int, int) { return counters() + std::max(kv4_rows_workspace(D), kv4_prompt_workspace(D)); }

int launch_kv4_attn(const Kv4Attn & a, int D, int type, void * ws, cudaStream_t st) {
    int * words = (int *) ws;
    void * parts = (char *) ws + counters();
    const int64_t most = std::min<int64_t>(a.max_q, a.n_tokens) * a.group;
    if (most <= KV4_FEW_ROWS) return launch_kv4_attn_rows(a, D, type, KV4_FEW_ROWS, words, parts, st);
    // a single sequence is not few, as far as the host can tell; of several, each goes where its rows belong
    const int few = a.n_seq > 1 ? KV4_FEW_ROWS : 0;
    if (few) {
        const int e = launch_kv4_attn_rows(a, D, type, few, words, parts, st);
        if (e) return e;
    }
    return launch_kv4_attn_prompt(a, D, type, few, words + KV4_COUNTERS, parts, st);
}

}  // namespace pb
