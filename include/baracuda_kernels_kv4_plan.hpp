// Typed plans of the attention step over the paged 4-bit cache (formulas, storage and statuses: baracuda_kernels_q.h), in the
// manner of baracuda_kernels_q_plan.hpp: descriptor and args per plan, select / workspace_size / run, typed errors, buffer lengths
// checked before a launch.
//
// Header-only; link against libbaracuda_kernels_q.so.
#pragma once

#include <cmath>
#include <initializer_list>
#include <vector>

#include "baracuda_kernels_q_plan.hpp"

namespace baracuda {

// A bf16 matrix: `len` elements from `ptr` on, rows `ld` elements apart.
template <typename T>
struct MatrixSpan {
    T* ptr = nullptr;
    size_t len = 0;
    int64_t ld = 0;
};

// One layer's cache.
struct Kv4CacheDescriptor {
    int32_t num_pages = 0, page_size = 0, heads_kv = 0, head_dim = 0;
    size_t page_bytes() const { return baracuda_kernels_kv4_page_bytes(page_size, heads_kv, head_dim); }
};

// The cache's buffer: `len` bytes from `ptr` on, pages `page_stride` bytes apart.
template <typename T>
struct Kv4CacheSpan {
    T* ptr = nullptr;
    size_t len = 0;
    int64_t page_stride = 0;
};

namespace detail {
template <typename T>
inline Error check_matrix(const MatrixSpan<T>& m, int64_t rows, int64_t cols) {
    if (m.ptr == nullptr || m.ld < cols) return Error::InvalidProblem;
    return m.len < span_elems(rows, cols, m.ld) ? Error::BufferTooSmall : Error::Ok;
}
template <typename T>
inline Error check_cache(const Kv4CacheSpan<T>& s, const Kv4CacheDescriptor& c) {
    if (s.ptr == nullptr || s.page_stride < static_cast<int64_t>(c.page_bytes())) return Error::InvalidProblem;
    return s.len < span_elems(c.num_pages, static_cast<int64_t>(c.page_bytes()), s.page_stride) ? Error::BufferTooSmall : Error::Ok;
}
inline Error first_of(std::initializer_list<Error> errors) {
    for (Error e : errors)
        if (e != Error::Ok) return e;
    return Error::Ok;
}
}  // namespace detail

// ---------------------------------------------------------------------------- norms, rotation, append
// rot_dim < 0: all of head_dim; 0: none.  axis_of_pair: empty, or the position axis of each of the rot_dim / 2 pairs.
struct QkNormRopeDescriptor {
    int32_t tokens = 0, heads_q = 0, heads_kv = 0, head_dim = 0;
    int32_t rot_dim = -1;
    bool interleaved = false;
    std::vector<uint8_t> axis_of_pair;
    float eps = 1e-6f;
    std::optional<Kv4CacheDescriptor> cache;  // keys and values go there instead of to k_out
};
struct QkNormRopeArgs {
    MatrixSpan<const void> q, k, v;
    DeviceSpan<const float> q_weight, k_weight;  // [head_dim], or none
    DeviceSpan<const float> cos_sin;             // [max_pos][rot_dim]
    int32_t max_pos = 0;
    DeviceSpan<const int32_t> positions;         // [axes][pos_stride]
    int64_t pos_stride = 0;
    MatrixSpan<void> q_out, k_out;
    Kv4CacheSpan<void> cache;
    DeviceSpan<const int64_t> slots;
};

class QkNormRopePlan {
  public:
    static Error select(const QkNormRopeDescriptor& desc, const PlanPreference& pref, QkNormRopePlan* out) {
        if (!detail::backend_ok(pref)) return Error::Unsupported;
        QkNormRopeDescriptor d = desc;
        if (d.rot_dim < 0) d.rot_dim = d.head_dim;
        int32_t axes = 1;
        if (!d.axis_of_pair.empty()) {
            if (d.axis_of_pair.size() != static_cast<size_t>(d.rot_dim) / 2) return Error::InvalidProblem;
            for (uint8_t a : d.axis_of_pair) {
                if (a > 7) return Error::InvalidProblem;
                axes = a >= axes ? a + 1 : axes;
            }
        }
        int32_t st;
        if (d.cache) {
            if (d.cache->heads_kv != d.heads_kv || d.cache->head_dim != d.head_dim || d.cache->num_pages < 0) return Error::InvalidProblem;
            st = baracuda_kernels_qk_norm_rope_kv4_append_bf16_sm100a_can_implement(d.tokens, d.heads_q, d.heads_kv, d.head_dim, d.rot_dim,
                                                                                    axes, d.cache->page_size);
        } else {
            st = baracuda_kernels_qk_norm_rope_bf16_sm100a_can_implement(d.tokens, d.heads_q, d.heads_kv, d.head_dim, d.rot_dim, axes);
        }
        if (st != 0) return status_to_error(st);
        out->desc_ = d;
        out->axes_ = axes;
        return Error::Ok;
    }
    size_t workspace_size() const { return 0; }
    Error run(void* stream, const QkNormRopeArgs& a) const {
        const QkNormRopeDescriptor& d = desc_;
        if (d.tokens == 0) return Error::Ok;
        const int64_t cols_q = static_cast<int64_t>(d.heads_q) * d.head_dim, cols = static_cast<int64_t>(d.heads_kv) * d.head_dim;
        Error e = detail::check_matrix(a.k, d.tokens, cols);
        if (e == Error::Ok && d.heads_q > 0)
            e = detail::first_of({detail::check_matrix(a.q, d.tokens, cols_q), detail::check_matrix(a.q_out, d.tokens, cols_q)});
        if (e != Error::Ok) return e;
        const size_t dim = static_cast<size_t>(d.head_dim);
        if ((a.q_weight.ptr != nullptr && a.q_weight.len < dim) || (a.k_weight.ptr != nullptr && a.k_weight.len < dim)) return Error::BufferTooSmall;
        if (d.rot_dim > 0) {
            if (a.cos_sin.ptr == nullptr || a.positions.ptr == nullptr || a.max_pos < 1) return Error::InvalidProblem;
            if (a.cos_sin.len < static_cast<size_t>(a.max_pos) * d.rot_dim) return Error::BufferTooSmall;
            if ((axes_ > 1 && a.pos_stride < d.tokens) || a.positions.len < detail::span_elems(axes_, d.tokens, a.pos_stride)) return Error::BufferTooSmall;
        }
        const uint8_t* table = d.axis_of_pair.empty() ? nullptr : d.axis_of_pair.data();
        if (!d.cache) {
            e = detail::check_matrix(a.k_out, d.tokens, cols);
            if (e != Error::Ok) return e;
            return status_to_error(baracuda_kernels_qk_norm_rope_bf16_sm100a_run(
                d.tokens, d.heads_q, d.heads_kv, d.head_dim, a.q.ptr, a.q.ld, a.k.ptr, a.k.ld, a.q_weight.ptr, a.k_weight.ptr, d.eps,
                a.cos_sin.ptr, d.rot_dim, a.max_pos, d.interleaved, a.positions.ptr, a.pos_stride, axes_, table, a.q_out.ptr, a.q_out.ld,
                a.k_out.ptr, a.k_out.ld, nullptr, 0, stream));
        }
        e = detail::first_of({detail::check_matrix(a.v, d.tokens, cols), detail::check_cache(a.cache, *d.cache)});
        if (e != Error::Ok) return e;
        if (a.slots.len < static_cast<size_t>(d.tokens)) return Error::BufferTooSmall;
        return status_to_error(baracuda_kernels_qk_norm_rope_kv4_append_bf16_sm100a_run(
            d.tokens, d.heads_q, d.heads_kv, d.head_dim, a.q.ptr, a.q.ld, a.k.ptr, a.k.ld, a.v.ptr, a.v.ld, a.q_weight.ptr, a.k_weight.ptr,
            d.eps, a.cos_sin.ptr, d.rot_dim, a.max_pos, d.interleaved, a.positions.ptr, a.pos_stride, axes_, table, a.q_out.ptr, a.q_out.ld,
            a.cache.ptr, a.cache.page_stride, d.cache->num_pages, d.cache->page_size, a.slots.ptr, nullptr, 0, stream));
    }

  private:
    QkNormRopeDescriptor desc_;
    int32_t axes_ = 1;
};

struct Kv4TokensDescriptor {
    int32_t tokens = 0;
    Kv4CacheDescriptor cache;
};

// Keys and values into the cache as they are.
class Kv4AppendPlan {
  public:
    static Error select(const Kv4TokensDescriptor& desc, const PlanPreference& pref, Kv4AppendPlan* out) {
        if (!detail::backend_ok(pref)) return Error::Unsupported;
        const Kv4CacheDescriptor& c = desc.cache;
        const int32_t st = baracuda_kernels_kv4_append_bf16_sm100a_can_implement(desc.tokens, c.heads_kv, c.head_dim, c.page_size);
        if (st != 0 || c.num_pages < 0) return st != 0 ? status_to_error(st) : Error::InvalidProblem;
        out->desc_ = desc;
        return Error::Ok;
    }
    size_t workspace_size() const { return 0; }
    Error run(void* stream, MatrixSpan<const void> k, MatrixSpan<const void> v, Kv4CacheSpan<void> cache, DeviceSpan<const int64_t> slots) const {
        const Kv4CacheDescriptor& c = desc_.cache;
        if (desc_.tokens == 0) return Error::Ok;
        const int64_t cols = static_cast<int64_t>(c.heads_kv) * c.head_dim;
        const Error e = detail::first_of({detail::check_matrix(k, desc_.tokens, cols), detail::check_matrix(v, desc_.tokens, cols),
                                          detail::check_cache(cache, c)});
        if (e != Error::Ok) return e;
        if (slots.len < static_cast<size_t>(desc_.tokens)) return Error::BufferTooSmall;
        return status_to_error(baracuda_kernels_kv4_append_bf16_sm100a_run(desc_.tokens, c.heads_kv, c.head_dim, k.ptr, k.ld, v.ptr, v.ld,
                                                                           cache.ptr, cache.page_stride, c.num_pages, c.page_size, slots.ptr,
                                                                           nullptr, 0, stream));
    }

  private:
    Kv4TokensDescriptor desc_;
};

// The tokens at `slots` as bf16.
class Kv4ReadPlan {
  public:
    static Error select(const Kv4TokensDescriptor& desc, const PlanPreference& pref, Kv4ReadPlan* out) {
        if (!detail::backend_ok(pref)) return Error::Unsupported;
        const Kv4CacheDescriptor& c = desc.cache;
        const int32_t st = baracuda_kernels_kv4_read_bf16_sm100a_can_implement(desc.tokens, c.heads_kv, c.head_dim, c.page_size);
        if (st != 0 || c.num_pages < 0) return st != 0 ? status_to_error(st) : Error::InvalidProblem;
        out->desc_ = desc;
        return Error::Ok;
    }
    size_t workspace_size() const { return 0; }
    Error run(void* stream, Kv4CacheSpan<const void> cache, DeviceSpan<const int64_t> slots, MatrixSpan<void> k, MatrixSpan<void> v) const {
        const Kv4CacheDescriptor& c = desc_.cache;
        if (desc_.tokens == 0) return Error::Ok;
        const int64_t cols = static_cast<int64_t>(c.heads_kv) * c.head_dim;
        const Error e = detail::first_of({detail::check_matrix(k, desc_.tokens, cols), detail::check_matrix(v, desc_.tokens, cols),
                                          detail::check_cache(cache, c)});
        if (e != Error::Ok) return e;
        if (slots.len < static_cast<size_t>(desc_.tokens)) return Error::BufferTooSmall;
        return status_to_error(baracuda_kernels_kv4_read_bf16_sm100a_run(desc_.tokens, c.heads_kv, c.head_dim, cache.ptr, cache.page_stride,
                                                                         c.num_pages, c.page_size, slots.ptr, k.ptr, k.ld, v.ptr, v.ld, nullptr,
                                                                         0, stream));
    }

  private:
    Kv4TokensDescriptor desc_;
};

// ---------------------------------------------------------------------------- attention
// max_q and max_kv bound the rows and cached tokens of any sequence; window > 0 lets a row see that many keys back, its own
// included.
struct Kv4AttentionDescriptor {
    int32_t batch = 0, max_q = 0, max_kv = 0, heads_q = 0;
    Kv4CacheDescriptor cache;
    bool causal = true;
    int32_t window = 0;
    std::optional<float> scale = std::nullopt;  // head_dim ** -0.5
};
struct Kv4AttentionArgs {
    int32_t total_q = 0;
    MatrixSpan<const void> q;
    DeviceSpan<const int32_t> cu_q, kv_lens;
    DeviceSpan<const int32_t> page_table;  // [batch][ld_table]
    int64_t ld_table = 0;
    Kv4CacheSpan<const void> cache;
    MatrixSpan<void> out;
    DeviceSpan<float> lse;  // [total_q][heads_q], or none
};

class Kv4AttentionPlan {
  public:
    static Error select(const Kv4AttentionDescriptor& desc, const PlanPreference& pref, Kv4AttentionPlan* out) {
        if (!detail::backend_ok(pref)) return Error::Unsupported;
        const Kv4CacheDescriptor& c = desc.cache;
        const int32_t st = baracuda_kernels_attention_kv4_bf16_sm100a_can_implement(desc.batch, desc.max_q, desc.max_kv, desc.heads_q, c.heads_kv,
                                                                                    c.head_dim, c.page_size);
        if (st != 0) return status_to_error(st);
        const float scale = desc.scale ? *desc.scale : 1.0f / std::sqrt(static_cast<float>(c.head_dim));
        if (c.num_pages < 0 || desc.window < 0 || !std::isfinite(scale)) return Error::InvalidProblem;
        const size_t bytes = baracuda_kernels_attention_kv4_bf16_sm100a_workspace_size(desc.batch, desc.max_q, desc.max_kv, desc.heads_q,
                                                                                       c.heads_kv, c.head_dim);
        if (bytes > pref.max_workspace_bytes) return Error::Unsupported;
        out->desc_ = desc;
        out->scale_ = scale;
        out->workspace_ = bytes;
        return Error::Ok;
    }
    size_t workspace_size() const { return workspace_; }
    Error run(void* stream, Workspace ws, const Kv4AttentionArgs& a) const {
        const Kv4AttentionDescriptor& d = desc_;
        const Kv4CacheDescriptor& c = d.cache;
        if (a.total_q < 0) return Error::InvalidProblem;
        if (d.batch == 0 || d.max_q == 0 || a.total_q == 0) return Error::Ok;
        const int64_t cols = static_cast<int64_t>(d.heads_q) * c.head_dim, pages = (static_cast<int64_t>(d.max_kv) + c.page_size - 1) / c.page_size;
        const Error e = detail::first_of({detail::check_matrix(a.q, a.total_q, cols), detail::check_matrix(a.out, a.total_q, cols),
                                          d.max_kv > 0 ? detail::check_cache(a.cache, c) : Error::Ok});
        if (e != Error::Ok) return e;
        if (a.cu_q.len < static_cast<size_t>(d.batch) + 1 || a.kv_lens.len < static_cast<size_t>(d.batch)) return Error::BufferTooSmall;
        if (a.ld_table < pages) return Error::InvalidProblem;
        if (a.page_table.len < detail::span_elems(d.batch, pages, a.ld_table)) return Error::BufferTooSmall;
        if (a.lse.ptr != nullptr && a.lse.len < static_cast<size_t>(a.total_q) * d.heads_q) return Error::BufferTooSmall;
        if (ws.bytes < workspace_) return Error::WorkspaceTooSmall;
        return status_to_error(baracuda_kernels_attention_kv4_bf16_sm100a_run(
            d.batch, a.total_q, d.max_q, d.max_kv, d.heads_q, c.heads_kv, c.head_dim, a.q.ptr, a.q.ld, a.cu_q.ptr, a.cache.ptr,
            a.cache.page_stride, c.num_pages, c.page_size, a.page_table.ptr, a.ld_table, a.kv_lens.ptr, scale_, d.causal, d.window, a.out.ptr,
            a.out.ld, a.lse.ptr, ws.ptr, ws.bytes, stream));
    }

  private:
    Kv4AttentionDescriptor desc_;
    float scale_ = 0.0f;
    size_t workspace_ = 0;
};

}  // namespace baracuda
