// Writing into a paged cache: new tokens to their pages and to the ring of queries, and whole pages to other pages.  Both move bytes and
// compute nothing: 16 bytes per lane, several loads ahead of their stores, and (HBM rewards long runs) a wavefront on neighbouring bytes.
#include "decode.hpp"

namespace mta {
namespace {

struct append_args {
    const char *x[3];           // new keys, values, queries: (slot, head, token, element), strides in 16-byte vectors
    int64_t batch[3], head[3], token[3];
    char *k, *v, *q;
    const int *table, *state;
    int64_t n_pages;
    int slots, max_pages, page_shift, heads, kv_heads, ring, tokens, vecs;   // vecs: 16-byte vectors of a row
};

// A workgroup writes one token of all heads of one slot's keys, values or queries (blockIdx.y).  What is read lies token by token (projections) or
// head by head, what is written head by head: lanes run along a row, then over the heads, so that reads of the former kind are one run and
// writes whole rows of 128 to 512 bytes either way.  Prompts of 4 x 1k to 4k tokens, 32 heads of 128 in 16 bits, us: one token per workgroup
// and two vectors per lane 59, eight and four 73 (more in flight is slower); with non-temporal stores 55.
template <bool STREAM> __global__ __launch_bounds__(256) void cache_append_kernel(const append_args a)
{
    const int b = blockIdx.z, what = blockIdx.y, tok = blockIdx.x, had = a.state[b], got = a.state[a.slots + b];
    const int count = got < a.tokens ? got : a.tokens;
    // (of the queries, the newest ones stay)
    if (had < 0 || tok >= count || (what == 2 && tok < count - a.ring)) return;
    const int64_t at = (int64_t)had + tok;
    const int total = (what == 2 ? a.heads : a.kv_heads) * a.vecs;
    const u32x4 *const x = reinterpret_cast<const u32x4 *>(a.x[what]) + b * a.batch[what] + tok * a.token[what];
    u32x4 *dst = reinterpret_cast<u32x4 *>(what == 0 ? a.k : what == 1 ? a.v : a.q);
    int64_t head;               // vectors between the rows of two heads
    if (what == 2) {
        head = (int64_t)a.ring * a.vecs;
        dst += (int64_t)b * a.heads * head + at % a.ring * a.vecs;
    } else {
        if ((at >> a.page_shift) >= a.max_pages) return;
        const int entry = a.table[(int64_t)b * a.max_pages + (at >> a.page_shift)];
        if ((unsigned)entry >= (uint64_t)a.n_pages) return;   // (a token without a page is dropped)
        head = (int64_t)a.vecs << a.page_shift;
        dst += (int64_t)entry * a.kv_heads * head + (at & ((1 << a.page_shift) - 1)) * a.vecs;
    }
    for (int i0 = threadIdx.x; i0 < total; i0 += 512) {
        u32x4 val[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int i = i0 + 256 * u, h = i / a.vecs;
            if (i < total) val[u] = x[h * a.head[what] + (i - h * a.vecs)];
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int i = i0 + 256 * u, h = i / a.vecs;
            if (i < total) {
                if constexpr (STREAM) __builtin_nontemporal_store(val[u], dst + h * head + (i - h * a.vecs));
                else dst[h * head + (i - h * a.vecs)] = val[u];
            }
        }
    }
}

constexpr int PAIRS = 480;
struct copy_args {
    char *pool[2];
    int64_t vecs;               // 16-byte vectors of a page
    int2 pair[PAIRS];
};
static_assert(sizeof(copy_args) <= 4096, "arguments of a launch");

// A workgroup moves 8 KB of one page of one pool.  The pairs travel as arguments: no copy to the device, nothing to wait for.  1000 pages of 2 x 128 KB,
// us, at 240 pairs a launch: two vectors per lane 96, four 105, eight 158 (as for reading, more in flight is slower); non-temporal stores 82.  480 pairs a
// launch, three launches in place of five: 88 with ordinary stores, 74 with non-temporal ones.
template <bool STREAM> __global__ __launch_bounds__(256) void cache_copy_pages_kernel(const copy_args a)
{
    const int2 pair = a.pair[blockIdx.y];
    char *const pool = a.pool[blockIdx.z];
    const u32x4 *const src = reinterpret_cast<const u32x4 *>(pool) + pair.x * a.vecs;
    u32x4 *const dst = reinterpret_cast<u32x4 *>(pool) + pair.y * a.vecs;
    const int64_t i0 = (int64_t)blockIdx.x * 512 + threadIdx.x;
    u32x4 val[2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
        if (i0 + 256 * u < a.vecs) val[u] = src[i0 + 256 * u];
#pragma unroll
    for (int u = 0; u < 2; ++u)
        if (i0 + 256 * u < a.vecs) {
            if constexpr (STREAM) __builtin_nontemporal_store(val[u], dst + i0 + 256 * u);
            else dst[i0 + 256 * u] = val[u];
        }
}

}  // namespace
}  // namespace mta

using namespace mta;

extern "C" int mta_cache_append(const mta_cache *c, const void *xq, const void *xk, const void *xv, const int64_t *strides, int64_t tokens, void *stream)
{
    if (const int e = check_cache(c)) return e;
    if (!xq || !xk || !xv || !strides) return MTA_ERR_NULL;
    if (tokens < 1 || tokens >= 1 << 24) return MTA_ERR_SHAPE;   // (a launch has fewer than 2^32 threads)
    const int size = dtype_size(c->dtype), per = 16 / size;
    append_args a = {};
    const void *xs[3] = {xk, xv, xq};
    for (int i = 0; i < 3; ++i) {
        const int64_t *s = strides + 3 * (i == 2 ? 0 : i + 1);   // (strides come in the order of the tensors: queries, keys, values)
        if (!aligned_to(xs[i], 16) || s[0] % per || s[1] % per || s[2] % per) return MTA_ERR_ALIGN;
        a.x[i] = (const char *)xs[i], a.batch[i] = s[0] / per, a.head[i] = s[1] / per, a.token[i] = s[2] / per;
    }
    a.k = (char *)c->k, a.v = (char *)c->v, a.q = (char *)c->q, a.table = c->table, a.state = c->state;
    a.n_pages = c->n_pages, a.slots = c->slots, a.max_pages = c->max_pages, a.page_shift = page_shift_of(c->page);
    a.heads = c->heads, a.kv_heads = c->kv_heads, a.ring = c->query_rows, a.tokens = (int)tokens, a.vecs = c->head_dim * size / 16;
    const hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)tokens, 3, (unsigned)c->slots);
    // (more than the caches keep for who reads the cache next)
    if (2 * tokens * c->slots * c->kv_heads * c->head_dim * size > 128 << 20) hipLaunchKernelGGL(cache_append_kernel<true>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(cache_append_kernel<false>, grid, dim3(256), 0, st, a);
    return launch_status();
}

extern "C" int mta_cache_copy_pages(void *k, void *v, int64_t n_pages, int64_t page_bytes, const int32_t *pairs, int64_t n, void *stream)
{
    if (!k || !v || (n > 0 && !pairs)) return MTA_ERR_NULL;
    if (n_pages <= 0 || n_pages > INT32_MAX || page_bytes <= 0 || page_bytes >= ((int64_t)1 << 36) || n < 0) return MTA_ERR_SHAPE;
    if (!aligned_to(k, 16) || !aligned_to(v, 16) || page_bytes % 16) return MTA_ERR_ALIGN;
    for (int64_t i = 0; i < 2 * n; ++i)
        if (pairs[i] < 0 || pairs[i] >= n_pages) return MTA_ERR_SHAPE;
    int64_t moves = 0;
    for (int64_t i = 0; i < n; ++i) moves += pairs[2 * i] != pairs[2 * i + 1];
    if (moves == 0) return MTA_OK;
    copy_args a;
    a.pool[0] = (char *)k, a.pool[1] = (char *)v, a.vecs = page_bytes / 16;
    const int64_t launches = (moves + PAIRS - 1) / PAIRS, each = (moves + launches - 1) / launches, chunks = (a.vecs + 511) / 512;
    const bool stream_out = 2 * moves * page_bytes > 128 << 20;   // (more than the caches keep for who reads the pages next)
    for (int64_t i = 0; moves > 0;) {
        int count = 0;
        for (; count < each && count < moves; ++i)
            if (pairs[2 * i] != pairs[2 * i + 1]) a.pair[count++] = make_int2(pairs[2 * i], pairs[2 * i + 1]);
        moves -= count;
        const dim3 grid((unsigned)chunks, (unsigned)count, 2);
        if (stream_out) hipLaunchKernelGGL(cache_copy_pages_kernel<true>, grid, dim3(256), 0, (hipStream_t)stream, a);
        else hipLaunchKernelGGL(cache_copy_pages_kernel<false>, grid, dim3(256), 0, (hipStream_t)stream, a);
        if (const int e = launch_status()) return e;
    }
    return MTA_OK;
}
