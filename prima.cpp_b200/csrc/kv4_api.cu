// prima.cpp_b200/csrc/kv4_api.cu — entry points of the 4-bit cache (include/prima_b200.h): checks of arguments in front of the launches.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <new>
#include <vector>

#include "../../include/prima_b200.h"
#include "kv4.cuh"

using namespace pb;

extern std::atomic<uint64_t> g_launches;

namespace {

int64_t page_bytes(const pb200_kv4_cache * c) { return (int64_t) c->n_layer * c->n_head_kv * kv4_chunk_bytes(c->head_dim); }
// 0, or why there is no such cache
int check(const pb200_kv4_cache * c) {
    if (!c || !c->pages || ((uintptr_t) c->pages & 15) || c->n_pages <= 0 || c->n_pages > INT32_MAX || c->n_layer <= 0 || c->n_head_kv <= 0) return PB200_EINVAL;
    if (!kv4_dim_ok(c->head_dim)) return PB200_ENOTSUP;
    if ((int64_t) c->n_layer * c->n_head_kv > 65535) return PB200_ENOTSUP;   // chunks of a page: an index of the grid
    return 0;
}
Kv4 layer_of(const pb200_kv4_cache * c, int layer) {
    return Kv4{(uint8_t *) c->pages + (int64_t) layer * c->n_head_kv * kv4_chunk_bytes(c->head_dim), page_bytes(c), c->n_pages, c->n_head_kv};
}
int elem_bytes(int type) { return type == PB200_TYPE_F32 ? 4 : type == PB200_TYPE_F16 || type == PB200_TYPE_BF16 ? 2 : 0; }
// rows of n numbers of a type: four at a time are loaded and stored
bool rows_ok(const void * p, int64_t ld, int64_t n, int eb) { return p && ((uintptr_t) p & (4 * eb - 1)) == 0 && ld >= n && ld % 4 == 0; }
// n rows of wa numbers every lda, n of wb every ldb (as rows_ok has them): whether they have a number in common.  With equal strides rows may lie between each other, as in a joint buffer
// (row j of b against row i of a: what counts is j - i); with others, ranges have to lie apart.
bool overlap(const void * a, int64_t lda, int64_t wa, const void * b, int64_t ldb, int64_t wb, int64_t n, int eb) {
    const int64_t at = (int64_t) ((uintptr_t) b - (uintptr_t) a), ld = lda * eb, end_a = (n - 1) * ld + wa * eb, end_b = (n - 1) * ldb * eb + wb * eb;
    if (end_a <= at || at + end_b <= 0) return false;
    if (lda != ldb) return true;
    const int64_t in = (at % ld + ld) % ld;     // where rows of b begin in a's stride
    return in < wa * eb || in + wb * eb > ld;
}

int attend(const pb200_kv4_cache * c, int layer, int type, const void * q, int64_t ldq, void * out, int64_t ldo, int n_head, int n_seq, const int32_t * q_start, const int32_t * kv_len,
           const int32_t * table, int64_t table_ld, int64_t n_tokens, int max_q, float scale, int window, int keep_first, float * lse, int64_t ld_lse, const Kv4Groups * groups, void * ws,
           size_t ws_bytes, void * stream) {
    const int e = check(c);
    if (e) return e;
    const int eb = elem_bytes(type);
    const int64_t D = c->head_dim;
    if (!eb || layer < 0 || layer >= c->n_layer || n_head <= 0 || n_head % c->n_head_kv || n_seq < 0 || n_tokens < 0 || n_tokens > INT32_MAX || max_q < 0) return PB200_EINVAL;
    if (!q_start || !kv_len || !table || table_ld <= 0 || !std::isfinite(scale) || window < 0 || keep_first < 0) return PB200_EINVAL;
    if (!rows_ok(q, ldq, n_head * D, eb) || !rows_ok(out, ldo, n_head * D, eb)) return PB200_EINVAL;
    if (lse && (((uintptr_t) lse & 3) || ld_lse < n_head)) return PB200_EINVAL;
    const size_t least = groups ? pb200_kv4_attn_shared_workspace_bytes(n_head, c->n_head_kv, c->head_dim, n_tokens) : pb200_kv4_attn_workspace_bytes(n_head, c->n_head_kv, c->head_dim);
    if (!ws || ((uintptr_t) ws & 15) || ws_bytes < least) return PB200_EINVAL;
    if (n_seq == 0 || n_tokens == 0 || max_q == 0) return 0;
    // what the kernels count in 31 bits: pages of all sequences, heads and tiles of eight rows where rows are few, tiles of all prompts otherwise
    const double group = n_head / c->n_head_kv, rows = std::min(std::min<double>(max_q, (double) n_tokens) * group, (double) KV4_FEW_ROWS);
    const auto pages_of = [&](int64_t ld) { return (double) std::min<int64_t>(ld, INT32_MAX / PB200_KV4_CELLS) * c->n_head_kv; };
    const double pages = n_seq * (pages_of(table_ld) + (groups ? pages_of(groups->table_ld) : 0.0)) * std::ceil(rows / 8);
    const double tiles = ((double) n_tokens * group / 128 + std::max(n_seq, groups ? groups->n : 0)) * c->n_head_kv;
    if (pages >= 2147483648.0 || tiles >= 2147483648.0 || n_tokens * group >= 2147483648.0) return PB200_ENOTSUP;
    if (overlap(q, ldq, n_head * D, out, ldo, n_head * D, n_tokens, eb)) return PB200_EINVAL;
    Kv4Attn a{layer_of(c, layer), q, ldq, out, ldo, n_head, n_head / c->n_head_kv, n_seq, q_start, kv_len, table, table_ld, n_tokens, max_q, window, keep_first, scale};
    a.x.lse = lse;
    a.x.ld_lse = ld_lse;
    int launches = 0;
    const int rc = groups ? launch_kv4_attn_shared(a, *groups, c->head_dim, type, ws, (cudaStream_t) stream, launches) : launch_kv4_attn(a, c->head_dim, type, ws, (cudaStream_t) stream, launches);
    g_launches += launches;
    return rc;
}

}  // namespace

extern "C" {

size_t pb200_kv4_page_bytes(int n_layer, int n_head_kv, int head_dim) {
    return n_layer > 0 && n_head_kv > 0 && kv4_dim_ok(head_dim) ? (size_t) n_layer * n_head_kv * kv4_chunk_bytes(head_dim) : 0;
}

int pb200_kv4_append(const pb200_kv4_cache * c, int layer, int type, const void * q, int64_t ldq, void * q_out, int64_t ldq_out, const void * k, int64_t ldk, const void * v,
                     int64_t ldv, int64_t n_tokens, int n_head, const int64_t * cells, const int32_t * pos, const float * q_norm, const float * k_norm, float eps,
                     const pb200_rope_args * rope, void * stream) {
    const int e = check(c);
    if (e) return e;
    const int eb = elem_bytes(type);
    const int64_t D = c->head_dim, kd = c->n_head_kv * D;
    if (!eb || layer < 0 || layer >= c->n_layer || n_tokens < 0 || n_tokens > 1 << 30 || n_head < 0 || !cells) return PB200_EINVAL;
    if (!rows_ok(k, ldk, kd, eb) || !rows_ok(v, ldv, kd, eb)) return PB200_EINVAL;
    if (n_head > 0 && (!rows_ok(q, ldq, n_head * D, eb) || !rows_ok(q_out, ldq_out, n_head * D, eb))) return PB200_EINVAL;
    if ((((uintptr_t) q_norm | (uintptr_t) k_norm) & 15) || ((q_norm || k_norm) && !(eps >= 0.f))) return PB200_EINVAL;
    if (n_head > 0 && n_tokens > 0) {   // rows that are read must not be another row's result: in place, or apart
        const auto over = [&](const void * p, int64_t ld, int64_t n) { return overlap(p, ld, n, q_out, ldq_out, n_head * D, n_tokens, eb); };
        if ((over(q, ldq, n_head * D) && !(q == q_out && ldq == ldq_out)) || over(k, ldk, kd) || over(v, ldv, kd)) return PB200_EINVAL;
    }
    Kv4Rope r{};
    if (rope && rope->n_dims != 0) {
        if (!pos || rope->n_dims < 0 || rope->n_dims > D || (rope->mode != 0 && rope->mode != 2) || !(rope->freq_base > 0.f) || !(rope->freq_scale > 0.f)) return PB200_EINVAL;
        if (rope->n_dims % 8) return PB200_ENOTSUP;
        // angle of pair i: pos * base^(-2 i / n) / factor, slowed down by freq_scale where the YaRN ramp (of pairs that turn too few times in the trained context) says so
        RopeParams y;
        rope_params_init(y, rope->n_dims, rope->mode, rope->n_ctx_orig, rope->freq_base, rope->freq_scale, rope->ext_factor, rope->attn_factor, rope->beta_fast, rope->beta_slow);
        r.n_dims = rope->n_dims;
        r.mode = rope->mode;
        r.freq_factors = rope->freq_factors;
        r.mscale = rope->attn_factor;
        if (rope->ext_factor != 0.f) r.mscale *= 1.0f + 0.1f * logf(1.0f / rope->freq_scale);
        for (int i = 0; i < rope->n_dims / 2; i++) {
            double mix = 0.0;
            if (rope->ext_factor != 0.f)
                mix = (1.0 - std::min(1.0, std::max(0.0, ((double) i - y.corr_dims[0]) / std::max(0.001, (double) y.corr_dims[1] - y.corr_dims[0])))) * rope->ext_factor;
            r.w[i] = std::pow((double) rope->freq_base, -2.0 * i / rope->n_dims) * ((double) rope->freq_scale * (1.0 - mix) + mix);
        }
    }
    if (n_tokens == 0) return 0;
    g_launches++;
    return launch_kv4_append(layer_of(c, layer), c->head_dim, type, q, ldq, q_out, ldq_out, k, ldk, v, ldv, n_tokens, n_head, cells, pos, n_head > 0 ? q_norm : nullptr, k_norm, eps, r,
                             (cudaStream_t) stream);
}

int pb200_kv4_load(const pb200_kv4_cache * c, int layer, int type, const int64_t * cells, int64_t n, void * k, int64_t ldk, void * v, int64_t ldv, void * stream) {
    const int e = check(c);
    if (e) return e;
    const int eb = elem_bytes(type);
    const int64_t kd = (int64_t) c->n_head_kv * c->head_dim;
    if (!eb || layer < 0 || layer >= c->n_layer || !cells || n < 0 || n > INT32_MAX || (!k && !v)) return PB200_EINVAL;
    if ((k && !rows_ok(k, ldk, kd, eb)) || (v && !rows_ok(v, ldv, kd, eb))) return PB200_EINVAL;
    if (n * kd / 4 / 256 >= INT32_MAX) return PB200_EINVAL;
    if (n == 0) return 0;
    g_launches++;
    return launch_kv4_load(layer_of(c, layer), c->head_dim, type, cells, n, k, ldk, v, ldv, (cudaStream_t) stream);
}

size_t pb200_kv4_attn_workspace_bytes(int n_head, int n_head_kv, int head_dim) {
    return n_head > 0 && n_head_kv > 0 && n_head % n_head_kv == 0 && kv4_dim_ok(head_dim) ? kv4_attn_workspace(head_dim) : 0;
}

int pb200_kv4_attn(const pb200_kv4_cache * c, int layer, int type, const void * q, int64_t ldq, void * out, int64_t ldo, int n_head, int n_seq, const int32_t * q_start,
                   const int32_t * kv_len, const int32_t * table, int64_t table_ld, int64_t n_tokens, int max_q, float scale, int window, int keep_first, void * ws,
                   size_t ws_bytes, void * stream) {
    return attend(c, layer, type, q, ldq, out, ldo, n_head, n_seq, q_start, kv_len, table, table_ld, n_tokens, max_q, scale, window, keep_first, nullptr, 0, nullptr, ws, ws_bytes, stream);
}

int pb200_kv4_attn_lse(const pb200_kv4_cache * c, int layer, int type, const void * q, int64_t ldq, void * out, int64_t ldo, int n_head, int n_seq, const int32_t * q_start,
                       const int32_t * kv_len, const int32_t * table, int64_t table_ld, int64_t n_tokens, int max_q, float scale, int window, int keep_first, float * lse, int64_t ld_lse,
                       void * ws, size_t ws_bytes, void * stream) {
    if (!lse) return PB200_EINVAL;
    return attend(c, layer, type, q, ldq, out, ldo, n_head, n_seq, q_start, kv_len, table, table_ld, n_tokens, max_q, scale, window, keep_first, lse, ld_lse, nullptr, ws, ws_bytes, stream);
}

size_t pb200_kv4_attn_shared_workspace_bytes(int n_head, int n_head_kv, int head_dim, int64_t n_tokens) {
    if (!pb200_kv4_attn_workspace_bytes(n_head, n_head_kv, head_dim) || n_tokens < 0 || n_tokens > INT32_MAX) return 0;
    return kv4_attn_shared_workspace(n_tokens * n_head, head_dim);
}

int pb200_kv4_attn_shared(const pb200_kv4_cache * c, int layer, int type, const void * q, int64_t ldq, void * out, int64_t ldo, int n_head, int n_seq, const int32_t * q_start,
                          const int32_t * kv_len, const int32_t * table, int64_t table_ld, int n_group, const int32_t * group_start, const int32_t * prefix_len, const int32_t * prefix_table,
                          int64_t prefix_ld, int64_t n_tokens, int max_q, float scale, float * lse, int64_t ld_lse, void * ws, size_t ws_bytes, void * stream) {
    if (n_group < 0 || (n_group > 0 && (!group_start || !prefix_len || !prefix_table || prefix_ld <= 0))) return PB200_EINVAL;
    if (n_group > 1 << 24) return PB200_ENOTSUP;      // (a group's number and a cell of a page in 31 bits)
    const Kv4Groups g{n_group, group_start, prefix_len, prefix_table, prefix_ld};
    return attend(c, layer, type, q, ldq, out, ldo, n_head, n_seq, q_start, kv_len, table, table_ld, n_tokens, max_q, scale, 0, 0, lse, ld_lse, n_group > 0 ? &g : nullptr, ws, ws_bytes, stream);
}

int pb200_kv4_weigh(const pb200_kv4_cache * c, int layer, int type, const void * q, int64_t ldq, int n_head, int n_seq, const int32_t * q_start, const int32_t * kv_len, const int32_t * table,
                    int64_t table_ld, int64_t n_tokens, int max_q, float scale, int window, int keep_first, const float * lse, int64_t ld_lse, float decay, const float * old, int64_t ld_old,
                    float * sums, int64_t ld_sums, void * stream) {
    const int e = check(c);
    if (e) return e;
    const int eb = elem_bytes(type);
    const int64_t D = c->head_dim;
    if (!eb || layer < 0 || layer >= c->n_layer || n_head <= 0 || n_head % c->n_head_kv || n_seq < 0 || n_tokens < 0 || n_tokens > INT32_MAX || max_q < 0) return PB200_EINVAL;
    if (!q_start || !kv_len || !table || table_ld <= 0 || !std::isfinite(scale) || window < 0 || keep_first < 0 || !std::isfinite(decay)) return PB200_EINVAL;
    if (n_tokens > 0 && (!rows_ok(q, ldq, n_head * D, eb) || !lse || ((uintptr_t) lse & 3) || ld_lse < n_head)) return PB200_EINVAL;
    if (!sums || ((uintptr_t) sums & 3) || ld_sums <= 0 || (old && (((uintptr_t) old & 3) || ld_old < ld_sums))) return PB200_EINVAL;
    // a sum is read and written by the same thread: in place, or apart
    if (old && n_seq > 0 && !(old == sums && ld_old == ld_sums) && overlap(old, ld_old, ld_sums, sums, ld_sums, ld_sums, n_seq, 4)) return PB200_EINVAL;
    // what the kernels count in 31 bits: cells, pages of all sequences, rows, blocks of rows of all heads
    const double rows = std::min((double) max_q, (double) n_tokens) * (n_head / c->n_head_kv);
    if (ld_sums > INT32_MAX - 4096 || (double) n_seq * ((double) ld_sums / PB200_KV4_CELLS + 1) >= 2147483648.0 - 65536 || rows >= 2147483648.0 || (rows / 64 + 1) * c->n_head_kv >= 2147483648.0)
        return PB200_ENOTSUP;
    if (n_seq == 0) return 0;
    Kv4Attn a{layer_of(c, layer), q, ldq, nullptr, 0, n_head, n_head / c->n_head_kv, n_seq, q_start, kv_len, table, table_ld, n_tokens, max_q, window, keep_first, scale};
    const Kv4Weigh w{a, lse, ld_lse, decay, decay == 0.f ? nullptr : old, ld_old, sums, ld_sums};
    g_launches++;
    return launch_kv4_weigh(w, c->head_dim, type, (cudaStream_t) stream);
}

int pb200_kv4_copy_pages(const pb200_kv4_cache * c, const int32_t * src, const int32_t * dst, int n, void * stream) {
    const int e = check(c);
    if (e) return e;
    if (n < 0 || (n > 0 && (!src || !dst))) return PB200_EINVAL;
    try {
        std::vector<int32_t> s(src, src + n), d(dst, dst + n);
        std::sort(s.begin(), s.end());
        std::sort(d.begin(), d.end());
        if (n > 0 && (s[0] < 0 || s[n - 1] >= c->n_pages || d[0] < 0 || d[n - 1] >= c->n_pages)) return PB200_EINVAL;
        for (int i = 0; i < n; i++)   // a page is written once, and none that is written is read: the copies have no order
            if ((i > 0 && d[i] == d[i - 1]) || std::binary_search(s.begin(), s.end(), d[i])) return PB200_EINVAL;
    } catch (const std::bad_alloc &) {
        return PB200_ENOMEM;
    }
    if (n == 0) return 0;
    g_launches += (n + 255) / 256;
    return launch_kv4_copy_pages((uint8_t *) c->pages, page_bytes(c), src, dst, n, (cudaStream_t) stream);
}

int pb200_kv4_compact(const pb200_kv4_cache * c, int n_seq, const int32_t * table, int64_t table_ld, const int32_t * to, int64_t to_ld, const int32_t * index, int64_t index_ld,
                      const int32_t * count, int max_count, void * stream) {
    const int e = check(c);
    if (e) return e;
    if (n_seq < 0 || n_seq > 65535 || max_count < 0 || !table || table_ld <= 0 || !to || to_ld <= 0 || !index || index_ld < max_count || !count) return PB200_EINVAL;
    if (n_seq == 0 || max_count == 0) return 0;
    g_launches++;
    return launch_kv4_compact((uint8_t *) c->pages, c->n_pages, c->n_layer * c->n_head_kv, c->head_dim, n_seq, table, table_ld, to, to_ld, index, index_ld, count, max_count,
                              (cudaStream_t) stream);
}

}  // extern "C"
