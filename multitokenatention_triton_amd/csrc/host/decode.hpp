// The paged cache's native entry points: checks of what the kernels rely on, workspace, one call into libmta_hip.so.
#pragma once

#include "ops.hpp"

#include <vector>

namespace mta_host {

// The cache as the C ABI takes it.  Pools, ring, table and state are used as they lie (they are written, and captured graphs keep their
// addresses), so what is not contiguous is refused and not copied.
inline mta_cache cache_of(const Tensor &k, const Tensor &v, const Tensor &q, const Tensor &table, const Tensor &state)
{
    for (const Tensor *t : {&k, &v, &q, &table, &state}) {
        TORCH_CHECK(t->is_cuda(), "the cache lives on ", t->device(), ": the MTA kernels only run on an AMD GPU (there is no CPU path)");
        TORCH_CHECK_VALUE(t->is_contiguous() && t->device() == k.device(), "the tensors of a cache are contiguous and on one device");
    }
    TORCH_CHECK_VALUE(k.dim() == 4 && k.sizes() == v.sizes() && q.dim() == 4 && q.size(3) == k.size(3),
                      "a cache has k and v of (pages, key heads, rows, D) and q of (slots, heads, rows, D), got ", k.sizes(), ", ", v.sizes(), " and ", q.sizes());
    TORCH_CHECK_TYPE(k.scalar_type() == v.scalar_type() && k.scalar_type() == q.scalar_type(), "k, v and q of a cache share a dtype");
    TORCH_CHECK_VALUE(table.scalar_type() == at::kInt && table.dim() == 2 && table.size(0) == q.size(0) && state.scalar_type() == at::kInt && state.dim() == 2
                          && state.size(0) == 2 && state.size(1) == q.size(0),
                      "a cache has an int32 table of (slots, pages) and an int32 state of (2, slots), got ", table.sizes(), " and ", state.sizes());
    TORCH_CHECK_VALUE(k.numel() > 0 && q.numel() > 0 && table.numel() > 0 && q.size(1) % k.size(1) == 0 && std::max({q.size(0), q.size(1), q.size(2), k.size(2), table.size(1)}) < (1 << 30),
                      "a cache of ", k.size(1), " key heads, ", q.size(1), " query heads, ", q.size(0), " slots");
    mta_cache c = {};
    c.k = out_ptr(k), c.v = out_ptr(v), c.q = out_ptr(q);
    c.table = table.const_data_ptr<int32_t>(), c.state = state.const_data_ptr<int32_t>();
    c.n_pages = k.size(0), c.slots = (int32_t)q.size(0), c.max_pages = (int32_t)table.size(1), c.page = (int32_t)k.size(2);
    c.heads = (int32_t)q.size(1), c.kv_heads = (int32_t)k.size(1), c.head_dim = (int32_t)k.size(3), c.query_rows = (int32_t)q.size(2);
    c.dtype = code(k, "cache");
    return c;
}

inline int64_t checked(int64_t bytes, const char *what)
{
    if (bytes < 0) check((int)bytes, what);
    return bytes;
}

inline void check_decode_weight(const Tensor &w, const Tensor &k, const char *what)
{
    TORCH_CHECK_VALUE(w.device() == k.device(), what, " lives on ", w.device(), ", the cache on ", k.device());
}

inline void check_rows(const mta_cache &c, int64_t rows)
{
    TORCH_CHECK_VALUE(c.query_rows >= rows, "this module needs the newest ", rows, " queries of a sequence, the cache keeps ", c.query_rows);
}

inline Tensor conv_attn_decode(const Tensor &k, const Tensor &v, const Tensor &q, const Tensor &table, const Tensor &state, int64_t longest, const Tensor &w_,
                               std::optional<double> softmax_scale, int64_t window)
{
    const mta_cache c = cache_of(k, v, q, table, state);
    const c10::OptionalDeviceGuard guard(k.device());
    check_conv_weight(w_, c.heads);
    check_decode_weight(w_, k, "W");
    check_rows(c, w_.size(1));
    TORCH_CHECK_VALUE(window >= 0 && window < (1 << 30), "window must be 0 (all keys) or a number of keys, got ", window);
    const Tensor w = on_gpu(w_, "W");
    const int r = (int)w.size(1), s = (int)w.size(2);
    const double scale = softmax_scale ? *softmax_scale : 1.0 / std::sqrt((double)c.head_dim);
    const int64_t bytes = checked(mta_conv_attn_decode_workspace(&c, longest, r, s, (int)window), "mta_conv_attn_decode");
    Tensor o = at::empty({c.slots, c.heads, 1, c.head_dim}, k.options()), ws;
    if (bytes) ws = at::empty({bytes}, k.options().dtype(at::kByte));
    check(mta_conv_attn_decode(&c, ptr(w), out_ptr(o), bytes ? out_ptr(ws) : nullptr, bytes, longest, r, s, (int)window, (float)scale, code(w, "W"), stream_of(k)),
          "mta_conv_attn_decode");
    return o;
}

// Absent weights are the identity.
inline Tensor mta_decode_step(const Tensor &k, const Tensor &v, const Tensor &q, const Tensor &table, const Tensor &state, int64_t longest, const Tensor &conv_w,
                              const OptTensor &w_pre, const OptTensor &post_conv_w, const OptTensor &w_post, int64_t pre_group, int64_t post_group, int64_t window)
{
    const mta_cache c = cache_of(k, v, q, table, state);
    const c10::OptionalDeviceGuard guard(k.device());
    TORCH_CHECK_VALUE(window >= 0 && window < (1 << 30), "window must be 0 (all keys) or a number of keys, got ", window);
    check_conv_weight(conv_w, c.heads);
    if (post_conv_w) check_conv_weight(*post_conv_w, c.heads);
    if (w_pre) check_head_weight(*w_pre, c.heads);
    if (w_post) check_head_weight(*w_post, c.heads);
    // (one dtype for all four; a mix of them goes as fp32, which holds them all)
    at::ScalarType type = conv_w.scalar_type();
    for (const OptTensor *t : {&w_pre, &post_conv_w, &w_post})
        if (*t && (*t)->scalar_type() != type) type = at::kFloat;
    auto take = [&](const Tensor &t, const char *what) {
        check_decode_weight(t, k, what);
        code(t, what);
        return on_gpu(t, what).to(type);
    };
    auto take_some = [&](const OptTensor &t, const char *what) { return t ? OptTensor(take(*t, what)) : OptTensor(); };
    const Tensor w = take(conv_w, "the conv weight");
    const OptTensor pre = take_some(w_pre, "the head weight ahead of the softmax"), w2 = take_some(post_conv_w, "the conv weight behind the softmax"),
                    post = take_some(w_post, "the head weight behind the softmax");
    const int r = (int)w.size(1), s = (int)w.size(2), r2 = w2 ? (int)w2->size(1) : 1, s2 = w2 ? (int)w2->size(2) : 1;
    check_rows(c, r + r2 - 1);
    const double scale = 1.0 / std::sqrt((double)c.head_dim);
    const int64_t bytes = checked(mta_decode_workspace(&c, longest, r, s, r2, s2, (int)pre_group, (int)post_group, (int)window), "mta_decode");
    Tensor o = at::empty({c.slots, 1, c.heads, c.head_dim}, k.options());
    const Tensor ws = at::empty({bytes}, k.options().dtype(at::kByte));
    check(mta_decode(&c, ptr(w), ptr(pre), ptr(w2), ptr(post), out_ptr(o), out_ptr(ws), bytes, longest, r, s, r2, s2, (int)pre_group, (int)post_group, (int)window,
                     (float)scale, code(w, "weights"), stream_of(k)),
          "mta_decode");
    return o;
}

inline void cache_append(const Tensor &k, const Tensor &v, const Tensor &q, const Tensor &table, const Tensor &state, const Tensor &xq_, const Tensor &xk_,
                         const Tensor &xv_)
{
    const mta_cache c = cache_of(k, v, q, table, state);
    const c10::OptionalDeviceGuard guard(k.device());
    TORCH_CHECK_VALUE(xq_.dim() == 4 && xk_.dim() == 4 && xk_.sizes() == xv_.sizes() && xq_.size(0) == c.slots && xk_.size(0) == c.slots && xq_.size(1) == c.heads
                          && xk_.size(1) == c.kv_heads && xq_.size(2) == xk_.size(2) && xq_.size(3) == c.head_dim && xk_.size(3) == c.head_dim,
                      "new tokens are (", c.slots, ",", c.heads, ",n,", c.head_dim, ") queries and (", c.slots, ",", c.kv_heads, ",n,", c.head_dim,
                      ") keys and values, got ", xq_.sizes(), ", ", xk_.sizes(), " and ", xv_.sizes());
    if (xq_.size(2) == 0) return;
    Tensor xs[3] = {xq_, xk_, xv_};
    int64_t strides[9];
    const int64_t per = 16 / k.element_size();
    for (int i = 0; i < 3; ++i) {
        Tensor &x = xs[i];
        TORCH_CHECK_VALUE(x.device() == k.device(), "new tokens live on ", x.device(), ", the cache on ", k.device());
        TORCH_CHECK_TYPE(x.scalar_type() == k.scalar_type(), "new tokens of ", x.scalar_type(), " for a cache of ", k.scalar_type());
        // (rows of whole vectors are read where they lie, others are copied first)
        auto odd = [&](int d) { return x.size(d) > 1 && x.stride(d) % per != 0; };
        if (x.stride(3) != 1 || odd(0) || odd(1) || odd(2) || reinterpret_cast<uintptr_t>(ptr(x)) % 16) x = x.clone(at::MemoryFormat::Contiguous);
        for (int d = 0; d < 3; ++d) strides[3 * i + d] = x.size(d) > 1 ? x.stride(d) : 0;
    }
    check(mta_cache_append(&c, ptr(xs[0]), ptr(xs[1]), ptr(xs[2]), strides, xs[0].size(2), stream_of(k)), "mta_cache_append");
}

inline void cache_copy_pages(const Tensor &k, const Tensor &v, const Tensor &pairs)
{
    TORCH_CHECK_VALUE(k.is_contiguous() && v.is_contiguous() && k.device() == v.device() && k.dim() >= 2 && k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type(),
                      "the pools are contiguous, on one device, of one shape and dtype");
    TORCH_CHECK_VALUE(!pairs.is_cuda() && (pairs.scalar_type() == at::kInt || pairs.scalar_type() == at::kLong) && pairs.dim() == 2 && pairs.size(1) == 2,
                      "pairs of pages are an (n,2) int32 or int64 tensor in host memory, got ", pairs.sizes(), " ", pairs.scalar_type(), " on ", pairs.device());
    const int64_t n = pairs.size(0), pages = k.size(0);
    if (n == 0) return;
    const Tensor wide = pairs.to(at::kLong).contiguous();
    const int64_t *const p = wide.const_data_ptr<int64_t>();
    std::vector<int32_t> list(2 * n), targets;
    targets.reserve(n);
    for (int64_t i = 0; i < 2 * n; ++i) {
        TORCH_CHECK_VALUE(p[i] >= 0 && p[i] < pages, "pairs of pages name page ", p[i], ", there are 0 .. ", pages - 1);
        list[i] = (int32_t)p[i];
        if (i % 2 && list[i] != list[i - 1]) targets.push_back(list[i]);
    }
    std::sort(targets.begin(), targets.end());
    bool clash = std::adjacent_find(targets.begin(), targets.end()) != targets.end();
    for (int64_t i = 0; i < n && !clash; ++i) clash = list[2 * i] != list[2 * i + 1] && std::binary_search(targets.begin(), targets.end(), list[2 * i]);
    TORCH_CHECK_VALUE(!clash, "a page is the target of two pairs, or target of one and source of another");
    TORCH_CHECK(k.is_cuda(), "the pools live on ", k.device(), ": the MTA kernels only run on an AMD GPU (there is no CPU path)");
    const c10::OptionalDeviceGuard guard(k.device());
    check(mta_cache_copy_pages(out_ptr(k), out_ptr(v), pages, k.numel() / pages * k.element_size(), list.data(), n, stream_of(k)), "mta_cache_copy_pages");
}

}  // namespace mta_host
