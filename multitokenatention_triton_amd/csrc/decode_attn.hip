// Fused conv-attention of the newest token of each slot of a paged cache: one pass over the keys and values,
//   raw_i[k] = q_i . K_k where row i sees key k, else 0            (i = p - R + 1 .. p, the newest rows)
//   s[k]     = scale * sum_{r < R, t < S} w[r][t] raw_{p - R + 1 + r}[k + t - (S-1)/2]
//   o        = sum_k exp(s[k]) V_k / sum_k exp(s[k])               over the keys k that row p sees
// shared out over the keys and joined.  Scores, statistics, probabilities and sums stay in fp32; the result is rounded once.
#include "decode.hpp"

namespace mta {
namespace {

// The results of an item: per (item, head) a row of D sums, then {reference, sum of exponentials}.
__host__ __device__ __forceinline__ int64_t stats_offset(int64_t items, int64_t heads, int D) { return items * heads * D; }

template <typename T, int D, int NT, int GW>
__global__ __launch_bounds__(256, 2) void conv_attn_decode_kernel(const decode_args a)
{
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int CH = 64 * NT;
    const int tid = threadIdx.x, lane = tid & 63, groups = a.heads / GW, index = blockIdx.x / groups, h0 = (blockIdx.x - index * groups) * GW;
    const shares sh(a, 0, log2_of(CH), false, lane);
    const work_item it = item_of(sh, index, -1, lane);
    if (it.slot < 0) return;
    const slot_step s = it.s;
    const int b = it.slot;
    T *const out = (T *)a.o + ((int64_t)b * a.heads + h0) * D;
    if (s.n <= 0) {
        for (int x = tid; x < GW * D; x += 256) out[x] = from_float<T>(s.n < 0 ? __builtin_nanf("") : 0.0f);
        return;
    }
    const int beg = s.base + (index - it.first) * sh.per * CH, end = beg + sh.per * CH < s.n ? beg + sh.per * CH : s.n;
    page_map pages;
    pages.load(a, b, beg - halo_left(a.S), lane);

    using lanes = score_lanes<NT, GW>;
    const int rows = GW * a.R, right = a.S - 1 - (a.S - 1) / 2;
    const raw_layout l = raw_layout_of(rows, a.R, a.S, GW, D, (int)sizeof(T), NT, true);
    raw_scores<T, D, NT> sc(a, smem, l, pages, rows, h0 / a.share, s.n, end + right < s.n ? end + right : s.n);
    const int wave = sc.wave, sp = (a.S + 3) & ~3;
    const lanes me(lane);
    const float *const weights = reinterpret_cast<const float *>(smem + l.weights) + me.head * a.R * sp;
    float *const probs = reinterpret_cast<float *>(smem + l.probs) + wave * GW * 16 * NT;
    const float scale2 = a.scale * LOG2E;

    // K and V are always under way a step ahead
    value_rows<T, D, NT, GW> val;
    typename raw_scores<T, D, NT>::start st;
    sc.begin(st, beg, b, h0);
    sc.load_step(beg);
    val.load(a, sc.pages, sc.kvh, beg + wave * 16 * NT, s.lo, end, lane);
    val.clear();
    sc.finish(st, beg, b, h0, smem, l);

    float m = -INFINITY, sum = 0.0f;   // a lane's head: reference, and its own keys' sum
    auto advance = [&](int kb, int step, auto more) {
        const int first = kb + wave * 16 * NT;
        sc.score_step(kb, step);
        if constexpr (more.value) {
            sc.pages.reach(a, b, kb + CH, kb + 2 * CH + sc.hr < sc.limit ? kb + 2 * CH + sc.hr : sc.limit, lane);
            sc.load_step(kb + CH);
        }
        __syncthreads();
        float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        with_taps(a.S, [&](auto count) {
            for (int r = me.part; r < a.R; r += lanes::RG)
                taps4<decltype(count)::value>(c, sc.window(step, me.head * a.R + r, wave * 16 * NT + 4 * me.quad), weights + r * sp, a.S);
        });
        me.deal(c);
        float top = m;
        bool seen[lanes::VALUES];
#pragma unroll
        for (int u = 0; u < lanes::VALUES; ++u) {
            const int key = first + me.key + u;
            seen[u] = key >= s.lo && key < end;
            top = fmaxf(top, seen[u] ? c[u] * scale2 : -INFINITY);
        }
        top = lanes::reduce(top, [](float x, float y) { return fmaxf(x, y); });
        if (__any(top > m)) {
            const float fade = m < top ? exp2f(m - top) : 1.0f;
            m = top;
            sum *= fade;
#pragma unroll
            for (int g = 0; g < GW; ++g) {
                const float f = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(fade), g * lanes::QUADS));
#pragma unroll
                for (int u = 0; u < val.E; ++u) val.acc[g][u] *= f;
            }
        }
        // (no score but -inf so far: a reference of 0, so that such keys count 0 and not NaN)
        const float ref = m == -INFINITY ? 0.0f : m;
        float *const to = probs + me.head * 16 * NT + me.key;
#pragma unroll
        for (int u = 0; u < lanes::VALUES; ++u) {
            const float p = seen[u] ? __builtin_amdgcn_exp2f(fmaf(c[u], scale2, -ref)) : 0.0f;   // (one rounding: the reference's own cancels)
            if (me.owner) {
                sum += p;
                to[u] = p;
            }
        }
        wave_sync();
        val.multiply(probs, first, s.lo, end, lane);
        if constexpr (more.value) val.load(a, sc.pages, sc.kvh, first + CH, s.lo, end, lane);
        wave_sync();
    };
    // (the last step apart: a branch around the loads of the others would cost their order)
    int kb = beg, step = 0;
    for (; kb + CH < end; kb += CH, ++step) advance(kb, step, count_of<1>());
    advance(kb, step, count_of<0>());
    sum = lanes::reduce(sum, [](float x, float y) { return x + y; });

    // the four wavefronts' results, brought to one reference
    __syncthreads();
    float *const res = reinterpret_cast<float *>(smem + l.raw), *const ml = res + DECODE_WAVES * GW * D;
    val.store(res + wave * GW * D, lane);
    if (me.quad == 0 && me.part == 0) ml[(wave * GW + me.head) * 2] = m, ml[(wave * GW + me.head) * 2 + 1] = sum;
    __syncthreads();
    for (int x = tid; x < GW * D; x += 256) {
        const int g = x / D, d = x % D;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < DECODE_WAVES; ++w) top = fmaxf(top, ml[(w * GW + g) * 2]);
        const float ref = top == -INFINITY ? 0.0f : top;
        float o = 0.0f, total = 0.0f;
#pragma unroll
        for (int w = 0; w < DECODE_WAVES; ++w) {
            const float f = exp2f(ml[(w * GW + g) * 2] - ref);
            o = fmaf(f, res[(w * GW + g) * D + d], o);
            total = fmaf(f, ml[(w * GW + g) * 2 + 1], total);
        }
        if (it.count == 1) {
            out[x] = from_float<T>(o / total);
        } else {
            const int64_t at = (int64_t)index * a.heads + h0 + g;
            a.ws[at * D + d] = o;
            if (d == 0) {
                float *ml_out = a.ws + stats_offset(a.items, a.heads, D) + 2 * at;
                ml_out[0] = top, ml_out[1] = total;
            }
        }
    }
}

// The items of one (slot, head), brought to one reference and added up, always in the same order.  A lane takes four elements of every PARTS-th
// item; the first AHEAD of its items are on their way while the factors are formed (a call over 8 slots of up to 4k keys, 32 heads 26.0 -> 24.7 us).
template <typename T, int D>
__global__ __launch_bounds__(256) void conv_attn_join_kernel(const decode_args a, int shift)
{
    constexpr int PARTS = 1024 / D, AHEAD = 4;
    __shared__ __align__(16) float so[PARTS][D];
    __shared__ float factor[64];
    const int h = blockIdx.x, b = blockIdx.y, d = threadIdx.x % (D / 4) * 4, part = threadIdx.x / (D / 4), lane = threadIdx.x & 63;
    T *const out = (T *)a.o + ((int64_t)b * a.heads + h) * D;
    const shares sh(a, 0, shift, false, lane);
    const work_item it = item_of(sh, 0, b, lane);
    const int items = it.count;
    if (items == 1) return;   // (that item wrote the result)
    const int64_t at = (int64_t)it.first * a.heads + h, stride = (int64_t)a.heads * D;
    const float *o = a.ws + at * D + d;
    const float2 *ml = reinterpret_cast<const float2 *>(a.ws + stats_offset(a.items, a.heads, D)) + at;
    f32x4 first[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) first[u] = *reinterpret_cast<const f32x4 *>(o + (part + u * PARTS < items ? part + u * PARTS : 0) * stride);
    float top = -INFINITY;
    for (int i = lane; i < items; i += 64) top = fmaxf(top, ml[(int64_t)i * a.heads].x);
    top = wave_max(top);
    const float ref = top == -INFINITY ? 0.0f : top;
    float total = 0.0f;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    const auto add = [&](int i, const f32x4 &x) {
        const float f = factor[i];
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] = fmaf(f, x[e], sum[e]);
    };
    for (int i0 = 0; i0 < items; i0 += 64) {   // (factors of 64 items at a time; all wavefronts form the same ones)
        const float2 x = i0 + lane < items ? ml[(int64_t)(i0 + lane) * a.heads] : make_float2(-INFINITY, 0.0f);
        const float f = __builtin_amdgcn_exp2f(x.x - ref);
        total += f * x.y;
        __syncthreads();
        if (threadIdx.x < 64) factor[lane] = f;
        __syncthreads();
        const int most = items - i0 < 64 ? items - i0 : 64;
        int i = part;
        if (i0 == 0) {
#pragma unroll
            for (int u = 0; u < AHEAD; ++u, i += PARTS)
                if (i < most) add(i, first[u]);
        }
#pragma unroll 4
        for (; i < most; i += PARTS) add(i, *reinterpret_cast<const f32x4 *>(o + (i0 + i) * stride));
    }
    total = wave_sum(total);
    *reinterpret_cast<f32x4 *>(&so[part][d]) = sum;
    __syncthreads();
    if (threadIdx.x >= D) return;
    float all = 0.0f;
#pragma unroll
    for (int i = 0; i < PARTS; ++i) all += so[i][threadIdx.x];
    out[threadIdx.x] = from_float<T>(all / total);
}

struct plan { cut t; int gw, lds; };

// Keys per step, heads per workgroup, items.
int plan_of(const mta_cache *c, int64_t longest, int R, int S, int window, plan &p)
{
    const int size = dtype_size(c->dtype), share = c->heads / c->kv_heads;
    const int64_t span = span_of(longest, window, 1);
    for (p.gw = 4; p.gw >= 1; p.gw >>= 1) {
        if (share % p.gw) continue;
        int most = most_tiles(c->head_dim * size);
        while (most > 1 && raw_layout_of(p.gw * R, R, S, p.gw, c->head_dim, size, most, true).total > 80 << 10) most >>= 1;
        p.t = cut_of(span, c->slots, c->heads / p.gw, most, 512, true);
        p.lds = raw_layout_of(p.gw * R, R, S, p.gw, c->head_dim, size, p.t.nt, true).total;
        if (p.lds <= (p.gw == 1 ? 160 << 10 : 80 << 10)) return too_many(p.t, c->heads / p.gw) ? MTA_ERR_SHAPE : MTA_OK;
    }
    return MTA_ERR_KERNEL_SIZE;
}

template <typename T, int D, int NT, int GW> int launch(const decode_args &a, const plan &p, hipStream_t st)
{
    auto kern = conv_attn_decode_kernel<T, D, NT, GW>;
    if (const int e = allow_lds(kern, p.lds)) return e;
    hipLaunchKernelGGL(kern, dim3((unsigned)(a.items * (a.heads / GW))), dim3(256), p.lds, st, a);
    if (p.t.joined) hipLaunchKernelGGL((conv_attn_join_kernel<T, D>), dim3((unsigned)a.heads, (unsigned)a.slots), dim3(256), 0, st, a, log2_of(64 * NT));
    return launch_status();
}
template <typename T, int D, int GW> int launch_steps(const decode_args &a, const plan &p, hipStream_t st)
{
    constexpr int MOST = most_tiles(D * (int)sizeof(T));
    if constexpr (MOST >= 4)
        if (p.t.nt == 4) return launch<T, D, 4, GW>(a, p, st);
    if constexpr (MOST >= 2)
        if (p.t.nt == 2) return launch<T, D, 2, GW>(a, p, st);
    return launch<T, D, 1, GW>(a, p, st);
}
template <typename T, int D> int launch_heads(const decode_args &a, const plan &p, hipStream_t st)
{
    return p.gw == 4 ? launch_steps<T, D, 4>(a, p, st) : p.gw == 2 ? launch_steps<T, D, 2>(a, p, st) : launch_steps<T, D, 1>(a, p, st);
}

int check_args(const mta_cache *c, int64_t longest, int R, int S, int window)
{
    if (const int e = check_cache(c)) return e;
    if (R < 1 || S < 1 || R > MTA_MAX_FUSED_KERNEL_R || S > MTA_MAX_FUSED_KERNEL_S) return MTA_ERR_KERNEL_SIZE;
    if (longest < 1 || longest > (int64_t)c->max_pages * c->page || window < 0 || c->query_rows < R) return MTA_ERR_SHAPE;
    return MTA_OK;
}

}  // namespace
}  // namespace mta

using namespace mta;

extern "C" int64_t mta_conv_attn_decode_workspace(const mta_cache *c, int64_t longest, int R, int S, int window)
{
    if (const int e = check_args(c, longest, R, S, window)) return e;
    plan p;
    if (const int e = plan_of(c, longest, R, S, window, p)) return e;
    return !p.t.joined ? 0 : (stats_offset(p.t.items, c->heads, c->head_dim) + 2 * (int64_t)p.t.items * c->heads) * 4;
}

extern "C" int mta_conv_attn_decode(const mta_cache *c, const void *w, void *o, void *workspace, int64_t workspace_bytes, int64_t longest, int R, int S,
                                    int window, float scale, int w_dtype, void *stream)
{
    if (const int e = check_args(c, longest, R, S, window)) return e;
    if (!w || !o) return MTA_ERR_NULL;
    if (dtype_size(w_dtype) == 0) return MTA_ERR_DTYPE;
    if (!aligned_to(w, dtype_size(w_dtype)) || !aligned_to(o, dtype_size(c->dtype)) || !aligned_to(workspace, 16)) return MTA_ERR_ALIGN;
    plan p;
    if (const int e = plan_of(c, longest, R, S, window, p)) return e;
    const int64_t need = mta_conv_attn_decode_workspace(c, longest, R, S, window);
    if (need > 0 && (!workspace || workspace_bytes < need)) return MTA_ERR_WORKSPACE;
    decode_args a = args_of(c, w, R, S, 1, window, longest, scale, w_dtype);
    a.o = o, a.ws = (float *)workspace, a.target = p.t.target, a.least = p.t.least, a.items = p.t.items, a.gw = p.gw;
    const hipStream_t st = (hipStream_t)stream;
    MTA_DISPATCH_IO(c->dtype, return c->head_dim == 64 ? launch_heads<io_t, 64>(a, p, st) : launch_heads<io_t, 128>(a, p, st));
}
