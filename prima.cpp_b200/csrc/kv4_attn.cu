// prima.cpp_b200/csrc/kv4_attn.cu — attention over the 4-bit cache (kv4.cuh): which kernel takes a sequence.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "../../include/prima_b200.h"
#include "kv4_attn.cuh"

namespace pb {

// A sequence with up to so many rows (queries x heads of a group) goes to the kernel of few rows, which walks its pages once for every eight of them; the other one has tiles of 128 and
// 256 rows whatever there are.  us, 8 sequences of 4096 cells, 32 heads over 8, few rows / prompt: bf16, 20 rows 38.7 / 77.5, 32 48.3 / 78.0, 48 59.8 / 80.7; F32, 32 65.8 / 78.0,
// 48 85.6 / 80.3.  64 sequences of 1000 cells, bf16: 32 rows 84 / 120, 48 109 / 120.
constexpr int KV4_FEW_ROWS = 48, KV4_FEW_ROWS_F32 = 32;

// counters (rows: one per warp and slice, zero between calls), tickets and a word for each slot, then the parts of either kernel, which run one after the other
static size_t counters() { return (KV4_COUNTERS + 64 + KV4_SLOTS) * sizeof(int); }
size_t kv4_attn_workspace(int D, int, int) { return counters() + std::max(kv4_rows_workspace(D), kv4_prompt_workspace(D)); }

int launch_kv4_attn(const Kv4Attn & a, int D, int type, void * ws, cudaStream_t st) {
    int * words = (int *) ws;
    void * parts = (char *) ws + counters();
    const int64_t most = std::min<int64_t>(a.max_q, a.n_tokens) * a.group;
    const int few = type == PB200_TYPE_F32 ? KV4_FEW_ROWS_F32 : KV4_FEW_ROWS;
    if (most <= few) return launch_kv4_attn_rows(a, D, type, few, words, parts, st);
    if (a.n_seq == 1) return launch_kv4_attn_prompt(a, D, type, 0, words + KV4_COUNTERS, parts, st);   // a prompt, as far as the host can tell: whatever rows it has
    const int e = launch_kv4_attn_rows(a, D, type, few, words, parts, st);                             // of several, each goes where its rows belong
    if (e) return e;
    return launch_kv4_attn_prompt(a, D, type, few, words + KV4_COUNTERS, parts, st);
}

}  // namespace pb
