// Flat C symbols of the attention step over the 4-bit cache: argument checks, then the launchers of kv4_*.cu.

#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/baracuda_kernels_q.h"
#include "kv4_format.cuh"
#include "launch.h"

namespace {

using namespace bq;

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

bool dim_served(int32_t d) { return d == 64 || d == 128 || d == 256; }

// Shape checks that every symbol shares: 0, or the status to return.
int32_t heads_status(int64_t count, int32_t heads_kv, int32_t head_dim) {
    if (count < 0 || heads_kv < 1 || head_dim < 1) return BQ_STATUS_INVALID_PROBLEM;
    if (!dim_served(head_dim) || heads_kv > 65536) return BQ_STATUS_UNSUPPORTED;
    return BQ_STATUS_OK;
}
int32_t page_status(int32_t page_size) {
    if (page_size < 1) return BQ_STATUS_INVALID_PROBLEM;
    return page_size % KV4_TILE != 0 || page_size > 65536 ? BQ_STATUS_UNSUPPORTED : BQ_STATUS_OK;
}
int32_t rotation_status(int32_t tokens, int32_t heads_q, int32_t heads_kv, int32_t head_dim, int32_t rot_dim, int32_t axes) {
    const int32_t st = heads_status(tokens, heads_kv, head_dim);
    if (st != BQ_STATUS_OK) return st;
    if (heads_q < 0 || rot_dim < 0 || rot_dim > head_dim || axes < 1) return BQ_STATUS_INVALID_PROBLEM;
    if (heads_q > 65536 || rot_dim % 8 != 0 || axes > 8) return BQ_STATUS_UNSUPPORTED;
    return BQ_STATUS_OK;
}

// The cache as the kernels see it; 0 or a status.
int32_t cache_of(Kv4Cache* c, const void* base, int64_t page_stride, int32_t num_pages, int32_t page_size, int32_t heads_kv,
                 int32_t head_dim) {
    const int32_t st = page_status(page_size);
    if (st != BQ_STATUS_OK) return st;
    if (base == nullptr || num_pages < 0) return BQ_STATUS_INVALID_PROBLEM;
    if (page_stride < static_cast<int64_t>(baracuda_kernels_kv4_page_bytes(page_size, heads_kv, head_dim))) return BQ_STATUS_INVALID_PROBLEM;
    if (!aligned(base, 16) || page_stride % 16 != 0) return BQ_STATUS_MISALIGNED;
    c->base = static_cast<uint8_t*>(const_cast<void*>(base));
    c->page_stride = page_stride;
    c->num_pages = num_pages;
    c->page_size = page_size;
    c->heads_kv = heads_kv;
    c->head_dim = head_dim;
    return BQ_STATUS_OK;
}

// One matrix of `heads` heads per row: pitch, pointer and alignment (elements of 2 bytes).
int32_t rows_status(const void* p, int64_t ld, int64_t heads, int32_t head_dim, int bytes) {
    if (p == nullptr || ld < heads * head_dim) return BQ_STATUS_INVALID_PROBLEM;
    return !aligned(p, bytes) || (ld * 2) % bytes != 0 ? BQ_STATUS_MISALIGNED : BQ_STATUS_OK;
}

int32_t run_norm_rope(NormRopeDesc& g, void* stream) {
    int32_t st = rotation_status(g.tokens, g.heads_q, g.heads_kv, g.head_dim, g.rot_dim, g.axes);
    if (st != BQ_STATUS_OK) return st;
    if (g.to_cache) {
        Kv4Cache c;
        st = page_status(g.cache.page_size);
        if (st != BQ_STATUS_OK) return st;
        if (g.tokens == 0) return BQ_STATUS_OK;
        st = cache_of(&c, g.cache.base, g.cache.page_stride, g.cache.num_pages, g.cache.page_size, g.heads_kv, g.head_dim);
        if (st != BQ_STATUS_OK) return st;
        g.cache = c;
        if (g.slots == nullptr) return BQ_STATUS_INVALID_PROBLEM;
        if (!aligned(g.slots, 8)) return BQ_STATUS_MISALIGNED;
        st = rows_status(g.v, g.ldv, g.heads_kv, g.head_dim, 8);
    } else {
        if (g.tokens == 0) return BQ_STATUS_OK;
        st = rows_status(g.k_out, g.ldko, g.heads_kv, g.head_dim, 8);
    }
    if (st != BQ_STATUS_OK) return st;
    st = rows_status(g.k, g.ldk, g.heads_kv, g.head_dim, 8);
    if (st != BQ_STATUS_OK) return st;
    if (g.heads_q > 0) {
        st = rows_status(g.q, g.ldq, g.heads_q, g.head_dim, 8);
        if (st == BQ_STATUS_OK) st = rows_status(g.q_out, g.ldqo, g.heads_q, g.head_dim, 8);
        if (st != BQ_STATUS_OK) return st;
    }
    if ((g.q_weight != nullptr || g.k_weight != nullptr) && !(g.eps >= 0.0f && isfinite(g.eps))) return BQ_STATUS_INVALID_PROBLEM;
    if (!aligned(g.q_weight, 16) || !aligned(g.k_weight, 16)) return BQ_STATUS_MISALIGNED;
    if (g.rot_dim > 0) {
        if (g.cos_sin == nullptr || g.positions == nullptr || g.max_pos < 1 || (g.axes > 1 && g.pos_stride < g.tokens)) return BQ_STATUS_INVALID_PROBLEM;
        if (!aligned(g.cos_sin, 16) || !aligned(g.positions, 4)) return BQ_STATUS_MISALIGNED;
        if (g.axis_of_pair == nullptr) g.axes = 1;
        for (int i = 0; g.axis_of_pair != nullptr && i < g.rot_dim / 2; ++i)
            if (g.axis_of_pair[i] >= g.axes) return BQ_STATUS_INVALID_PROBLEM;
    }
    return launch_qk_norm_rope(g, static_cast<cudaStream_t>(stream));
}

}  // namespace

extern "C" {

size_t baracuda_kernels_kv4_page_bytes(int32_t page_size, int32_t heads_kv, int32_t head_dim) {
    if (heads_status(0, heads_kv, head_dim) != BQ_STATUS_OK || page_status(page_size) != BQ_STATUS_OK) return 0;
    return static_cast<size_t>(page_size / KV4_TILE) * heads_kv * kv4_tile_bytes(head_dim);
}

int32_t baracuda_kernels_qk_norm_rope_bf16_sm100a_can_implement(int32_t tokens, int32_t heads_q, int32_t heads_kv,
                                                                int32_t head_dim, int32_t rot_dim, int32_t axes) {
    return rotation_status(tokens, heads_q, heads_kv, head_dim, rot_dim, axes);
}
size_t baracuda_kernels_qk_norm_rope_bf16_sm100a_workspace_size(int32_t, int32_t, int32_t, int32_t) { return 0; }
int32_t baracuda_kernels_qk_norm_rope_bf16_sm100a_run(
    int32_t tokens, int32_t heads_q, int32_t heads_kv, int32_t head_dim, const void* q, int64_t ldq, const void* k, int64_t ldk,
    const void* q_weight, const void* k_weight, float eps, const void* cos_sin, int32_t rot_dim, int32_t max_pos,
    int32_t interleaved, const void* positions, int64_t pos_stride, int32_t axes, const uint8_t* axis_of_pair, void* q_out,
    int64_t ldqo, void* k_out, int64_t ldko, void*, size_t, void* stream) {
    NormRopeDesc g = {};
    g.tokens = tokens, g.heads_q = heads_q, g.heads_kv = heads_kv, g.head_dim = head_dim;
    g.q = q, g.ldq = ldq, g.k = k, g.ldk = ldk;
    g.q_weight = static_cast<const float*>(q_weight), g.k_weight = static_cast<const float*>(k_weight), g.eps = eps;
    g.cos_sin = static_cast<const float*>(cos_sin), g.rot_dim = rot_dim, g.max_pos = max_pos, g.interleaved = interleaved != 0;
    g.positions = static_cast<const int32_t*>(positions), g.pos_stride = pos_stride, g.axes = axes, g.axis_of_pair = axis_of_pair;
    g.q_out = q_out, g.ldqo = ldqo, g.k_out = k_out, g.ldko = ldko;
    return run_norm_rope(g, stream);
}

int32_t baracuda_kernels_qk_norm_rope_kv4_append_bf16_sm100a_can_implement(int32_t tokens, int32_t heads_q, int32_t heads_kv,
                                                                           int32_t head_dim, int32_t rot_dim, int32_t axes,
                                                                           int32_t page_size) {
    const int32_t st = rotation_status(tokens, heads_q, heads_kv, head_dim, rot_dim, axes);
    return st != BQ_STATUS_OK ? st : page_status(page_size);
}
size_t baracuda_kernels_qk_norm_rope_kv4_append_bf16_sm100a_workspace_size(int32_t, int32_t, int32_t, int32_t) { return 0; }
int32_t baracuda_kernels_qk_norm_rope_kv4_append_bf16_sm100a_run(
    int32_t tokens, int32_t heads_q, int32_t heads_kv, int32_t head_dim, const void* q, int64_t ldq, const void* k, int64_t ldk,
    const void* v, int64_t ldv, const void* q_weight, const void* k_weight, float eps, const void* cos_sin, int32_t rot_dim,
    int32_t max_pos, int32_t interleaved, const void* positions, int64_t pos_stride, int32_t axes, const uint8_t* axis_of_pair,
    void* q_out, int64_t ldqo, void* cache, int64_t page_stride, int32_t num_pages, int32_t page_size, const void* slots, void*,
    size_t, void* stream) {
    NormRopeDesc g = {};
    g.tokens = tokens, g.heads_q = heads_q, g.heads_kv = heads_kv, g.head_dim = head_dim;
    g.q = q, g.ldq = ldq, g.k = k, g.ldk = ldk, g.v = v, g.ldv = ldv;
    g.q_weight = static_cast<const float*>(q_weight), g.k_weight = static_cast<const float*>(k_weight), g.eps = eps;
    g.cos_sin = static_cast<const float*>(cos_sin), g.rot_dim = rot_dim, g.max_pos = max_pos, g.interleaved = interleaved != 0;
    g.positions = static_cast<const int32_t*>(positions), g.pos_stride = pos_stride, g.axes = axes, g.axis_of_pair = axis_of_pair;
    g.q_out = q_out, g.ldqo = ldqo;
    g.to_cache = 1;
    g.cache.base = static_cast<uint8_t*>(cache), g.cache.page_stride = page_stride, g.cache.num_pages = num_pages, g.cache.page_size = page_size;
    g.slots = static_cast<const int64_t*>(slots);
    return run_norm_rope(g, stream);
}

int32_t baracuda_kernels_kv4_append_bf16_sm100a_can_implement(int32_t tokens, int32_t heads_kv, int32_t head_dim, int32_t page_size) {
    const int32_t st = heads_status(tokens, heads_kv, head_dim);
    return st != BQ_STATUS_OK ? st : page_status(page_size);
}
size_t baracuda_kernels_kv4_append_bf16_sm100a_workspace_size(int32_t, int32_t, int32_t) { return 0; }
int32_t baracuda_kernels_kv4_append_bf16_sm100a_run(int32_t tokens, int32_t heads_kv, int32_t head_dim, const void* k, int64_t ldk,
                                                    const void* v, int64_t ldv, void* cache, int64_t page_stride, int32_t num_pages,
                                                    int32_t page_size, const void* slots, void*, size_t, void* stream) {
    NormRopeDesc g = {};
    g.tokens = tokens, g.heads_kv = heads_kv, g.head_dim = head_dim, g.axes = 1;
    g.k = k, g.ldk = ldk, g.v = v, g.ldv = ldv;
    g.to_cache = 1;
    g.cache.base = static_cast<uint8_t*>(cache), g.cache.page_stride = page_stride, g.cache.num_pages = num_pages, g.cache.page_size = page_size;
    g.slots = static_cast<const int64_t*>(slots);
    return run_norm_rope(g, stream);
}

int32_t baracuda_kernels_kv4_read_bf16_sm100a_can_implement(int32_t tokens, int32_t heads_kv, int32_t head_dim, int32_t page_size) {
    return baracuda_kernels_kv4_append_bf16_sm100a_can_implement(tokens, heads_kv, head_dim, page_size);
}
size_t baracuda_kernels_kv4_read_bf16_sm100a_workspace_size(int32_t, int32_t, int32_t) { return 0; }
int32_t baracuda_kernels_kv4_read_bf16_sm100a_run(int32_t tokens, int32_t heads_kv, int32_t head_dim, const void* cache,
                                                  int64_t page_stride, int32_t num_pages, int32_t page_size, const void* slots,
                                                  void* k, int64_t ldk, void* v, int64_t ldv, void*, size_t, void* stream) {
    int32_t st = baracuda_kernels_kv4_read_bf16_sm100a_can_implement(tokens, heads_kv, head_dim, page_size);
    if (st != BQ_STATUS_OK || tokens == 0) return st;
    Kv4ReadDesc g = {};
    st = cache_of(&g.cache, cache, page_stride, num_pages, page_size, heads_kv, head_dim);
    if (st == BQ_STATUS_OK) st = rows_status(k, ldk, heads_kv, head_dim, 16);
    if (st == BQ_STATUS_OK) st = rows_status(v, ldv, heads_kv, head_dim, 16);
    if (st == BQ_STATUS_OK && slots == nullptr) st = BQ_STATUS_INVALID_PROBLEM;
    if (st == BQ_STATUS_OK && !aligned(slots, 8)) st = BQ_STATUS_MISALIGNED;
    if (st != BQ_STATUS_OK) return st;
    g.tokens = tokens;
    g.slots = static_cast<const int64_t*>(slots);
    g.k = k, g.ldk = ldk, g.v = v, g.ldv = ldv;
    return launch_kv4_read(g, static_cast<cudaStream_t>(stream));
}

int32_t baracuda_kernels_attention_kv4_bf16_sm100a_can_implement(int32_t batch, int32_t max_q, int32_t max_kv, int32_t heads_q,
                                                                 int32_t heads_kv, int32_t head_dim, int32_t page_size) {
    int32_t st = heads_status(batch, heads_kv, head_dim);
    if (st == BQ_STATUS_OK) st = page_status(page_size);
    if (st != BQ_STATUS_OK) return st;
    if (max_q < 0 || max_kv < 0 || heads_q < 1 || heads_q % heads_kv != 0) return BQ_STATUS_INVALID_PROBLEM;
    // the kernels count blocks, rows of a kv head and keys in 32 bits
    if (heads_q > 65536 || max_kv > 0x7fff0000 || static_cast<int64_t>(max_q) * (heads_q / heads_kv) > 0x7fff0000) return BQ_STATUS_UNSUPPORTED;
    return kv4_attention_fits(batch, max_q, max_kv, heads_q, heads_kv, head_dim) ? BQ_STATUS_OK : BQ_STATUS_UNSUPPORTED;
}
size_t baracuda_kernels_attention_kv4_bf16_sm100a_workspace_size(int32_t batch, int32_t max_q, int32_t max_kv, int32_t heads_q,
                                                                 int32_t heads_kv, int32_t head_dim) {
    if (baracuda_kernels_attention_kv4_bf16_sm100a_can_implement(batch, max_q, max_kv, heads_q, heads_kv, head_dim, KV4_TILE) != BQ_STATUS_OK)
        return 0;
    if (batch == 0 || max_q == 0) return 0;
    return kv4_attention_workspace_bytes(batch, max_q, max_kv, heads_q, heads_kv, head_dim);
}
int32_t baracuda_kernels_attention_kv4_bf16_sm100a_run(
    int32_t batch, int32_t total_q, int32_t max_q, int32_t max_kv, int32_t heads_q, int32_t heads_kv, int32_t head_dim, const void* q,
    int64_t ldq, const void* cu_q, const void* cache, int64_t page_stride, int32_t num_pages, int32_t page_size,
    const void* page_table, int64_t ld_table, const void* kv_lens, float scale, int32_t causal, int32_t window, void* out,
    int64_t ldo, void* lse, void* workspace, size_t workspace_bytes, void* stream) {
    int32_t st = baracuda_kernels_attention_kv4_bf16_sm100a_can_implement(batch, max_q, max_kv, heads_q, heads_kv, head_dim, page_size);
    if (st != BQ_STATUS_OK) return st;
    if (total_q < 0 || window < 0 || !isfinite(scale)) return BQ_STATUS_INVALID_PROBLEM;
    if (batch == 0 || total_q == 0 || max_q == 0) return BQ_STATUS_OK;
    Kv4AttentionDesc g = {};
    if (cache == nullptr && max_kv == 0) {  // no key anywhere: nothing of the cache is read
        g.cache.page_size = page_size, g.cache.heads_kv = heads_kv, g.cache.head_dim = head_dim;
    } else {
        st = cache_of(&g.cache, cache, page_stride, num_pages, page_size, heads_kv, head_dim);
        if (st != BQ_STATUS_OK) return st;
    }
    st = rows_status(q, ldq, heads_q, head_dim, 16);
    if (st == BQ_STATUS_OK) st = rows_status(out, ldo, heads_q, head_dim, 16);
    if (st != BQ_STATUS_OK) return st;
    if (cu_q == nullptr || kv_lens == nullptr) return BQ_STATUS_INVALID_PROBLEM;
    if (max_kv > 0 && (page_table == nullptr || ld_table < (static_cast<int64_t>(max_kv) + page_size - 1) / page_size))
        return BQ_STATUS_INVALID_PROBLEM;
    if (!aligned(cu_q, 4) || !aligned(kv_lens, 4) || !aligned(page_table, 4) || !aligned(lse, 4)) return BQ_STATUS_MISALIGNED;
    const size_t need = kv4_attention_workspace_bytes(batch, max_q, max_kv, heads_q, heads_kv, head_dim);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return BQ_STATUS_WORKSPACE;
    if (need > 0 && !aligned(workspace, 16)) return BQ_STATUS_MISALIGNED;
    g.batch = batch, g.total_q = total_q, g.max_q = max_q, g.max_kv = max_kv, g.heads_q = heads_q;
    g.q = q, g.ldq = ldq, g.cu_q = static_cast<const int32_t*>(cu_q);
    g.page_table = static_cast<const int32_t*>(page_table), g.ld_table = ld_table, g.kv_lens = static_cast<const int32_t*>(kv_lens);
    g.scale = scale, g.causal = causal != 0, g.window = window;
    g.out = out, g.ldo = ldo, g.lse = static_cast<float*>(lse);
    g.workspace = workspace, g.workspace_bytes = workspace_bytes;
    return launch_kv4_attention(g, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
