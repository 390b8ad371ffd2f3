// Fused conv-attention of the newest token of each slot of a paged cache: one pass over the keys and values,
//   raw_i[k] = q_i . K_k where row i sees key k, else 0            (i = p - R + 1 .. p, the newest rows)
//   s[k]     = scale * sum_{r < R, t < S} w[r][t] raw_{p - R + 1 + r}[k + t - (S-1)/2]
//   o        = sum_k exp(s[k]) V_k / sum_k exp(s[k])               over the keys k that row p sees
// split over the keys and joined.  Scores, statistics, probabilities and sums stay in fp32; the result is rounded once.
#include "decode.hpp"

namespace mta {
namespace {

// The results of a split: per (slot, head, split) a row of D sums, then {reference, sum of exponentials}.
__host__ __device__ __forceinline__ int64_t stats_offset(int64_t slots, int64_t heads, int64_t splits, int D) { return slots * heads * splits * D; }

template <typename T, int D, int NT, int GW>
__global__ __launch_bounds__(256) void conv_attn_decode_kernel(const decode_args a)
{
    extern __shared__ __align__(16) unsigned char smem[];
    const int b = blockIdx.z, h0 = blockIdx.y * GW, split = blockIdx.x, tid = threadIdx.x;
    T *const out = (T *)a.o + ((int64_t)b * a.heads + h0) * D;
    const slot_step s = step_of(a, b, 0);
    if (s.n <= 0) {
        if (a.n_splits == 1)   // (else the join says so)
            for (int x = tid; x < GW * D; x += 256) out[x] = from_float<T>(s.n < 0 ? __builtin_nanf("") : 0.0f);
        return;
    }
    const int beg = s.base + split * a.split_len;
    if (beg >= s.n) return;
    const int end = beg + a.split_len < s.n ? beg + a.split_len : s.n;

    constexpr int CH = 64 * NT, QUADS = 4 * NT, SUBS = 64 / QUADS;   // (four keys per lane, a key's rows of taps dealt over SUBS lanes)
    const int rows = GW * a.R, left = (a.S - 1) / 2, reach = end + a.S - 1 - left;
    const raw_layout l = raw_layout_of(rows, a.R, a.S, GW, D, (int)sizeof(T), NT, true);
    raw_scores<T, D, NT> sc(a, smem, l, rows, b, h0 / a.share, s.n, reach < s.n ? reach : s.n);
    const int lane = sc.lane, wave = sc.wave, quad = lane % QUADS, sub = lane / QUADS, mine = 4 * quad + lane / 16;
    const bool owner = lane % 16 < QUADS;   // (with NT < 4 several lanes come to hold the same key)
    const float *const weights = reinterpret_cast<const float *>(smem + l.weights);
    float *const probs = reinterpret_cast<float *>(smem + l.probs) + wave * GW * 16 * NT;
    const int sp = (a.S + 3) & ~3;
    const float scale2 = a.scale * LOG2E;

    sc.load_step(beg);
    sc.stage(smem, l, b, h0);
    __syncthreads();
    sc.halo(beg);

    value_rows<T, D, NT, GW> val;
    val.clear();
    float m[GW], sum[GW];
#pragma unroll
    for (int g = 0; g < GW; ++g) m[g] = -INFINITY, sum[g] = 0.0f;

    int step = 0;
    for (int kb = beg; kb < end; kb += CH, ++step) {
        const int first = kb + wave * 16 * NT;
        val.load(first, s.lo, end, lane, [&](int key0) { return sc.tile(a.v, key0); });
        sc.score_step(kb, step);
        if (kb + CH < end) sc.load_step(kb + CH);
        __syncthreads();
        const int key = first + mine;
        const bool seen = key >= s.lo && key < end;
#pragma unroll
        for (int g = 0; g < GW; ++g) {
            float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            with_taps(a.S, [&](auto count) {
                for (int r = sub; r < a.R; r += SUBS)
                    taps4<decltype(count)::value>(part, sc.window(step, g * a.R + r, wave * 16 * NT + 4 * quad), weights + (g * a.R + r) * sp, a.S);
            });
            const float c = deal4<NT>(part);
            const float e = seen ? c * scale2 : -INFINITY;
            const float top = fmaxf(m[g], wave_max(e));
            if (top > m[g]) {   // (wavefront-uniform)
                const float fade = exp2f(m[g] - top);
                m[g] = top;
                sum[g] *= fade;
#pragma unroll
                for (int u = 0; u < val.E; ++u) val.acc[g][u] *= fade;
            }
            // (no score but -inf so far: a reference of 0, so that such keys count 0 and not NaN)
            const float p = seen ? __builtin_amdgcn_exp2f(e - (m[g] == -INFINITY ? 0.0f : m[g])) : 0.0f;
            if (owner) {
                sum[g] += p;
                probs[g * 16 * NT + mine] = p;
            }
        }
        wave_sync();
        val.multiply(probs, lane);
        wave_sync();
    }

    // the four wavefronts' results, brought to one reference
    __syncthreads();
    float *const res = reinterpret_cast<float *>(smem + l.raw), *const ml = res + DECODE_WAVES * GW * D;
    val.store(res + wave * GW * D, lane);
#pragma unroll
    for (int g = 0; g < GW; ++g) {
        const float total = wave_sum(sum[g]);
        if (lane == 0) ml[(wave * GW + g) * 2] = m[g], ml[(wave * GW + g) * 2 + 1] = total;
    }
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
        if (a.n_splits == 1) {
            out[x] = from_float<T>(o / total);
        } else {
            const int64_t at = ((int64_t)b * a.heads + h0 + g) * a.n_splits + split;
            a.ws[at * D + d] = o;
            if (d == 0) {
                float *st = a.ws + stats_offset(a.slots, a.heads, a.n_splits, D) + 2 * at;
                st[0] = top, st[1] = total;
            }
        }
    }
}

// The splits of one (slot, head), brought to one reference and added up, always in the same order.
template <typename T, int D>
__global__ __launch_bounds__(256) void conv_attn_join_kernel(const decode_args a)
{
    constexpr int PARTS = 256 / D;
    __shared__ float so[PARTS][D], factor[64];
    const int h = blockIdx.x, b = blockIdx.y, d = threadIdx.x % D, part = threadIdx.x / D, lane = threadIdx.x & 63;
    T *const out = (T *)a.o + ((int64_t)b * a.heads + h) * D;
    const slot_step s = step_of(a, b, 0);
    if (s.n <= 0) {
        if (part == 0) out[d] = from_float<T>(s.n < 0 ? __builtin_nanf("") : 0.0f);
        return;
    }
    const int splits = (s.n - s.base + a.split_len - 1) / a.split_len;
    const int64_t at = ((int64_t)b * a.heads + h) * a.n_splits;
    const float *o = a.ws + at * D;
    const float2 *ml = reinterpret_cast<const float2 *>(a.ws + stats_offset(a.slots, a.heads, a.n_splits, D)) + at;
    float top = -INFINITY;
    for (int i = lane; i < splits; i += 64) top = fmaxf(top, ml[i].x);
    top = wave_max(top);
    const float ref = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f, total = 0.0f;
    for (int i0 = 0; i0 < splits; i0 += 64) {   // (factors of 64 splits at a time; all wavefronts form the same ones)
        const float2 x = i0 + lane < splits ? ml[i0 + lane] : make_float2(-INFINITY, 0.0f);
        const float f = __builtin_amdgcn_exp2f(x.x - ref);
        total += f * x.y;
        __syncthreads();
        if (threadIdx.x < 64) factor[lane] = f;
        __syncthreads();
        const int most = splits - i0 < 64 ? splits - i0 : 64;
#pragma unroll 8
        for (int i = part; i < most; i += PARTS) sum = fmaf(factor[i], o[(int64_t)(i0 + i) * D + d], sum);
    }
    total = wave_sum(total);
    so[part][d] = sum;
    __syncthreads();
    if (part != 0) return;
#pragma unroll
    for (int i = 1; i < PARTS; ++i) sum += so[i][d];
    out[d] = from_float<T>(sum / total);
}

struct plan { int nt, gw, split_len, n_splits, lds; };

// Keys per step, heads per workgroup, keys per split.
int plan_of(const mta_cache *c, int64_t longest, int R, int S, int window, plan &p)
{
    const int size = dtype_size(c->dtype), share = c->heads / c->kv_heads, wide = c->head_dim * size > 256 ? 2 : 4;
    const int64_t span = span_of(longest, window, 1);
    for (int gw = 4; gw >= 1; gw >>= 1) {
        if (share % gw) continue;
        for (int nt = wide;; nt = 1) {
            const int lds = raw_layout_of(gw * R, R, S, gw, c->head_dim, size, nt, true).total;
            const int64_t steps = (span + 64 * nt - 1) / (64 * nt), groups = (int64_t)c->slots * (c->heads / gw);
            // (long steps only where they still make enough workgroups)
            if (lds <= (nt == 1 ? 160 << 10 : 80 << 10) && (nt == 1 || steps * groups >= 512)) {
                const int64_t per = (steps * groups + 1023) / 1024;
                p.nt = nt, p.gw = gw, p.lds = lds, p.split_len = (int)(per < steps ? per : steps) * 64 * nt;
                p.n_splits = (int)((span + p.split_len - 1) / p.split_len);
                return MTA_OK;
            }
            if (nt == 1) break;
        }
    }
    return MTA_ERR_KERNEL_SIZE;
}

template <typename T, int D, int NT, int GW> int launch(const decode_args &a, const plan &p, hipStream_t st)
{
    auto kern = conv_attn_decode_kernel<T, D, NT, GW>;
    if (const int e = allow_lds(kern, p.lds)) return e;
    hipLaunchKernelGGL(kern, dim3((unsigned)p.n_splits, (unsigned)(a.heads / GW), (unsigned)a.slots), dim3(256), p.lds, st, a);
    if (p.n_splits > 1) hipLaunchKernelGGL((conv_attn_join_kernel<T, D>), dim3((unsigned)a.heads, (unsigned)a.slots), dim3(256), 0, st, a);
    return launch_status();
}
template <typename T, int D, int NT> int launch_heads(const decode_args &a, const plan &p, hipStream_t st)
{
    return p.gw == 4 ? launch<T, D, NT, 4>(a, p, st) : p.gw == 2 ? launch<T, D, NT, 2>(a, p, st) : launch<T, D, NT, 1>(a, p, st);
}
template <typename T, int D> int launch_steps(const decode_args &a, const plan &p, hipStream_t st)
{
    constexpr int WIDE = D * (int)sizeof(T) > 256 ? 2 : 4;
    return p.nt == 1 ? launch_heads<T, D, 1>(a, p, st) : launch_heads<T, D, WIDE>(a, p, st);
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
    return p.n_splits == 1 ? 0 : (stats_offset(c->slots, c->heads, p.n_splits, c->head_dim) + 2 * (int64_t)c->slots * c->heads * p.n_splits) * 4;
}

extern "C" int mta_conv_attn_decode(const mta_cache *c, const void *w, void *o, void *workspace, int64_t workspace_bytes, int64_t longest, int R, int S,
                                    int window, float scale, int w_dtype, void *stream)
{
    if (const int e = check_args(c, longest, R, S, window)) return e;
    if (!w || !o) return MTA_ERR_NULL;
    if (dtype_size(w_dtype) == 0) return MTA_ERR_DTYPE;
    if (!aligned_to(w, dtype_size(w_dtype)) || !aligned_to(o, dtype_size(c->dtype)) || !aligned_to(workspace, 8)) return MTA_ERR_ALIGN;
    plan p;
    if (const int e = plan_of(c, longest, R, S, window, p)) return e;
    const int64_t need = mta_conv_attn_decode_workspace(c, longest, R, S, window);
    if (need > 0 && (!workspace || workspace_bytes < need)) return MTA_ERR_WORKSPACE;
    decode_args a = args_of(c, w, R, S, 1, window, longest, scale, w_dtype);
    a.o = o, a.ws = (float *)workspace, a.split_len = p.split_len, a.n_splits = p.n_splits, a.gw = p.gw;
    const hipStream_t st = (hipStream_t)stream;
    MTA_DISPATCH_IO(c->dtype, return c->head_dim == 64 ? launch_steps<io_t, 64>(a, p, st) : launch_steps<io_t, 128>(a, p, st));
}
