// Multi-Token Attention of the newest token of each slot of a paged cache.  With P the newest position, R x S and R2 x S2 the two conv
// kernels, and rows j = P - R2 + 1 .. P (the only ones that reach the newest row through the second conv):
//   raw_i[k] = scale * q_i . K_k where row i sees key k, else 0                       i = P - R2 - R + 2 .. P
//   s1_j[k]  = sum_{r, t} w[h][r][t] raw_{j - R + 1 + r}[k + t - (S-1)/2]              per head h
//   s2_j     = sum_g Wpre[h][g] s1_j (head g)                                         p_j = softmax over the keys that row j sees
//   p1[k]    = sum_{r, t} w2[h][r][t] p_{P - R2 + 1 + r}[k + t - (S2-1)/2]             p2 = sum_g Wpost[h][g] p1 (head g)
//   o        = sum_k p2[k] V_k
// Heads and rows meet between the stages, so this is not one pass but four or five short kernels around the two that stream: scores (K once),
// mixing with the rows' statistics, the second conv (none where it is the identity: a single row is left then), mixing and values (V once),
// and the sum over the splits.  What goes between them is R2 numbers of fp32 per key and head, against 2 D of K and V.
#include "decode.hpp"

namespace mta {
namespace {

struct mta_args {
    decode_args d;
    const void *w_pre, *w_post, *w2;
    int pre_group, post_group;  // heads that mix (1: the identity, no weight)
    int R2, S2, span;           // span: keys that a row of the workspace has room for
    int chunk, chunks;          // keys per workgroup of the mixing kernel
    int v_len, v_splits;        // keys per split of the values kernel
    float *s1, *s2, *p1, *part;
    float *stats;               // (slot, head, row, chunk): reference, sum of exponentials
};

__device__ __forceinline__ slot_step step_of(const mta_args &a, int b)
{
    return mta::step_of(a.d, b, a.R2 - 1);
}
// the keys that output row j sees: lo .. pos
__device__ __forceinline__ int row_pos(const mta_args &a, int n, int j) { return n - a.R2 + j; }
__device__ __forceinline__ bool sees(const mta_args &a, int pos, int key) { return key >= 0 && key <= pos && (a.d.window == 0 || key > pos - a.d.window); }

// ---- scores: K once ----
// R2 = 1: as in conv-attention a key's rows of taps are dealt over the lanes that share it.  Else the output rows are, JB to a lane: a window of
// raw scores is read once for all of them.
template <typename T, int D, int NT, int JB, bool ONE>
__global__ __launch_bounds__(256) void decode_scores_kernel(const mta_args m)
{
    extern __shared__ __align__(16) unsigned char smem[];
    const decode_args &a = m.d;
    const int b = blockIdx.z, h0 = blockIdx.y * a.gw, split = blockIdx.x;
    const slot_step s = step_of(m, b);
    if (s.n <= 0) return;
    const int beg = s.base + split * a.split_len;
    if (beg >= s.n) return;
    const int end = beg + a.split_len < s.n ? beg + a.split_len : s.n;

    constexpr int CH = 64 * NT, QUADS = 4 * NT, SUBS = 64 / QUADS;
    const int rows = a.gw * a.W, left = (a.S - 1) / 2, reach = end + a.S - 1 - left;
    const raw_layout l = raw_layout_of(rows, a.R, a.S, a.gw, D, (int)sizeof(T), NT, false);
    raw_scores<T, D, NT> sc(a, smem, l, rows, b, h0 / a.share, s.n, reach < s.n ? reach : s.n);
    const int lane = sc.lane, wave = sc.wave, quad = lane % QUADS, sub = lane / QUADS;
    const float *const weights = reinterpret_cast<const float *>(smem + l.weights);
    const int sp = (a.S + 3) & ~3;

    sc.load_step(beg);
    sc.stage(smem, l, b, h0);
    __syncthreads();
    sc.halo(beg);
    int step = 0;
    for (int kb = beg; kb < end; kb += CH, ++step) {
        sc.score_step(kb, step);
        if (kb + CH < end) sc.load_step(kb + CH);
        __syncthreads();
        const int local = wave * 16 * NT + 4 * quad, key = kb + local;
        float *const out = m.s1 + ((int64_t)b * a.heads + h0) * m.R2 * m.span + (key - s.base);
        for (int g = 0; g < a.gw; ++g) {
            const float *const w = weights + g * a.R * sp;
            if constexpr (ONE) {
                float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                with_taps(a.S, [&](auto count) {
                    for (int r = sub; r < a.R; r += SUBS)
                        taps4<decltype(count)::value>(part, sc.window(step, g * a.W + r, local), w + r * sp, a.S);
                });
                const float c = deal4<NT>(part);
                if (lane % 16 < QUADS && key + lane / 16 < end) out[(int64_t)g * m.span + lane / 16] = c * a.scale;
            } else {
                for (int j0 = sub * JB; j0 < m.R2; j0 += SUBS * JB) {
                    float c[JB][4];
#pragma unroll
                    for (int u = 0; u < JB; ++u) c[u][0] = c[u][1] = c[u][2] = c[u][3] = 0.0f;
                    with_taps(a.S, [&](auto count) {
                        for (int i = 0; i < a.R + JB - 1; ++i) {
                            // (behind the last row there are outputs that nobody writes)
                            const float *x = sc.window(step, g * a.W + (j0 + i < a.W ? j0 + i : a.W - 1), local);
#pragma unroll
                            for (int u = 0; u < JB; ++u)
                                if (i - u >= 0 && i - u < a.R) taps4<decltype(count)::value>(c[u], x, w + (i - u) * sp, a.S);   // (wavefront-uniform)
                        }
                    });
#pragma unroll
                    for (int u = 0; u < JB; ++u)   // (whole vectors: a row has room for them, and nobody reads behind the last key)
                        if (j0 + u < m.R2 && key < end)
                            *reinterpret_cast<f32x4 *>(out + ((int64_t)g * m.R2 + j0 + u) * m.span) = f32x4{c[u][0], c[u][1], c[u][2], c[u][3]} * a.scale;
                }
            }
        }
    }
}

// ---- mixing ahead of the softmax, and the statistics of the rows ----
// A wavefront takes blocks of four heads of a group, a lane a key of each 64; (reference, sum) run along per lane and meet at the end.
__global__ __launch_bounds__(256) void decode_mix_kernel(const mta_args m)
{
    extern __shared__ __align__(16) float lds[];
    const int b = blockIdx.z, j = blockIdx.y, chunk = blockIdx.x, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const slot_step s = step_of(m, b);
    if (s.n <= 0) return;
    const int k0 = s.base + chunk * m.chunk, pos = row_pos(m, s.n, j), H = m.d.heads, grp = m.pre_group;
    if (k0 >= s.n) return;
    const int end = k0 + m.chunk < s.n ? k0 + m.chunk : s.n, per = (grp + 3) / 4, blocks = H / grp * per;
    f32x4 *const w = reinterpret_cast<f32x4 *>(lds) + wave * grp;
    for (int blk = wave; blk < blocks; blk += 4) {
        const int g0 = blk / per * grp, o0 = g0 + (blk % per) * 4, cnt = g0 + grp - o0 < 4 ? g0 + grp - o0 : 4;
        if (m.w_pre) {
            wave_sync();
            for (int x = lane; x < grp * 4; x += 64)
                lds[wave * grp * 4 + x] = (x & 3) < cnt ? load_any(m.w_pre, m.d.w_dtype, (int64_t)(o0 + (x & 3)) * H + g0 + (x >> 2)) : 0.0f;
            wave_sync();
        }
        float top[4], sum[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) top[u] = -INFINITY, sum[u] = 0.0f;
        for (int kk = k0; kk < end; kk += 64) {
            const int key = kk + lane;
            const bool in = key < end, seen = in && sees(m, pos, key);
            f32x4 c = {0.0f, 0.0f, 0.0f, 0.0f};
            const float *x = m.s1 + (((int64_t)b * H + g0) * m.R2 + j) * m.span + (in ? key - s.base : 0);
            const int64_t head = (int64_t)m.R2 * m.span;
            if (m.w_pre) {
#pragma unroll 4
                for (int g = 0; g < grp; ++g) {
                    const float v = x[g * head];
                    const f32x4 wg = w[g];
#pragma unroll
                    for (int u = 0; u < 4; ++u) c[u] = fmaf(wg[u], v, c[u]);
                }
            } else {
                c[0] = x[0];   // (groups of one head)
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (u >= cnt) break;
                if (m.w_pre && in) m.s2[(((int64_t)b * H + o0 + u) * m.R2 + j) * m.span + (key - s.base)] = c[u];
                if (seen) {
                    const float e = c[u] * LOG2E, t = fmaxf(top[u], e), ref = t == -INFINITY ? 0.0f : t;
                    sum[u] = sum[u] * __builtin_amdgcn_exp2f(top[u] - ref) + __builtin_amdgcn_exp2f(e - ref);
                    top[u] = t;
                }
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (u >= cnt) break;
            const float t = wave_max(top[u]), ref = t == -INFINITY ? 0.0f : t;
            const float l = wave_sum(sum[u] * __builtin_amdgcn_exp2f(top[u] - ref));
            if (lane == 0) {
                float *st = m.stats + ((((int64_t)b * H + o0 + u) * m.R2 + j) * m.chunks + chunk) * 2;
                st[0] = t, st[1] = l;
            }
        }
    }
}

// {reference * log2(e), 1 / sum} of a row from its chunks; PARTS neighbouring lanes share a row
template <int PARTS> __device__ __forceinline__ float2 row_statistics(const float *st, int chunks, int part)
{
    float top = -INFINITY, sum = 0.0f;
    for (int c = part; c < chunks; c += PARTS) {
        const float2 x = *reinterpret_cast<const float2 *>(st + 2 * c);
        const float t = fmaxf(top, x.x), ref = t == -INFINITY ? 0.0f : t;
        sum = sum * __builtin_amdgcn_exp2f(top - ref) + x.y * __builtin_amdgcn_exp2f(x.x - ref);
        top = t;
    }
#pragma unroll
    for (int o = PARTS / 2; o >= 1; o >>= 1) {
        const float t2 = __shfl_xor(top, o), s2 = __shfl_xor(sum, o), t = fmaxf(top, t2), ref = t == -INFINITY ? 0.0f : t;
        sum = sum * __builtin_amdgcn_exp2f(top - ref) + s2 * __builtin_amdgcn_exp2f(t2 - ref);
        top = t;
    }
    return make_float2(top, 1.0f / sum);
}

// ---- the conv behind the softmax: probabilities of R2 rows of a head, one row out ----
__global__ __launch_bounds__(256) void decode_post_kernel(const mta_args m)
{
    extern __shared__ __align__(16) float lds[];
    const int b = blockIdx.z, h = blockIdx.y, tid = threadIdx.x;
    const slot_step s = step_of(m, b);
    if (s.n <= 0) return;
    const int k0 = s.base + blockIdx.x * 256;
    if (k0 >= s.n) return;
    const int left = (m.S2 - 1) / 2, cols = 256 + m.S2 - 1, taps = m.R2 * m.S2, H = m.d.heads;
    float2 *const stat = reinterpret_cast<float2 *>(lds);
    float *const w = lds + 2 * m.R2, *const p = w + taps;
    const int64_t row0 = ((int64_t)b * H + h) * m.R2;
    const int chunks = (s.n - s.base + m.chunk - 1) / m.chunk;
    for (int x = tid; x < m.R2 * 8; x += 256) {
        const float2 st = row_statistics<8>(m.stats + (row0 + x / 8) * m.chunks * 2, chunks, x % 8);
        if (x % 8 == 0) stat[x / 8] = st;
    }
    for (int x = tid; x < taps; x += 256) w[x] = load_any(m.w2, m.d.w_dtype, (int64_t)h * taps + x);
    __syncthreads();
    const float *const sc = m.w_pre ? m.s2 : m.s1;
    for (int j = 0; j < m.R2; ++j) {
        const int pos = row_pos(m, s.n, j);
        const float2 st = stat[j];
        for (int c = tid; c < cols; c += 256) {
            const int key = k0 + c - left;
            p[j * cols + c] = key >= s.base && sees(m, pos, key) ? __builtin_amdgcn_exp2f(sc[(row0 + j) * m.span + (key - s.base)] * LOG2E - st.x) * st.y : 0.0f;
        }
    }
    __syncthreads();
    const int key = k0 + tid;
    if (key >= s.n) return;
    float c = 0.0f;
    for (int j = 0; j < m.R2; ++j)
        for (int t = 0; t < m.S2; ++t) c = fmaf(w[j * m.S2 + t], p[j * cols + tid + t], c);
    m.p1[((int64_t)b * H + h) * m.span + (key - s.base)] = key >= s.lo ? c : 0.0f;
}

// ---- mixing behind the softmax and P V: V once ----
// POST: p1 has been through the second conv; else the heads' probabilities are formed here, from scores and statistics.
template <typename T, int D, int NT, int GW, bool POST>
__global__ __launch_bounds__(256) void decode_values_kernel(const mta_args m)
{
    extern __shared__ __align__(16) float lds[];
    const decode_args &a = m.d;
    const int b = blockIdx.z, h0 = blockIdx.y * GW, split = blockIdx.x, tid = threadIdx.x;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), H = a.heads, grp = m.post_group;
    T *const out = (T *)a.o + ((int64_t)b * H + h0) * D;
    const slot_step s = step_of(m, b);
    if (s.n <= 0) {
        if (m.v_splits == 1)
            for (int x = tid; x < GW * D; x += 256) out[x] = from_float<T>(s.n < 0 ? __builtin_nanf("") : 0.0f);
        return;
    }
    const int first_key = s.lo & ~15, beg = first_key + split * m.v_len;
    if (beg >= s.n) return;
    const int end = beg + m.v_len < s.n ? beg + m.v_len : s.n;

    constexpr int CH = 64 * NT, SUBS = 4 / NT;
    const int sub = lane / (16 * NT), mine = lane % (16 * NT);
    float2 *const coef = reinterpret_cast<float2 *>(lds);               // [GW][grp]: reference, weight / sum
    float *const probs = lds + 2 * GW * grp + wave * GW * 16 * NT;
    float *const res = lds + 2 * GW * grp + DECODE_WAVES * GW * 16 * NT;
    for (int x = tid; x < GW * grp * 8; x += 256) {
        const int g = x / 8 / grp, i = x / 8 - g * grp, from = (h0 + g) / grp * grp + i;
        float2 st = make_float2(0.0f, 1.0f);
        if constexpr (!POST) st = row_statistics<8>(m.stats + ((int64_t)b * H + from) * m.chunks * 2, (s.n - s.base + m.chunk - 1) / m.chunk, x % 8);
        if (x % 8 == 0) {
            if (m.w_post) st.y *= load_any(m.w_post, a.w_dtype, (int64_t)(h0 + g) * H + from);
            coef[x / 8] = st;
        }
    }
    __syncthreads();
    const int *const entries = a.table + (int64_t)b * a.max_pages;
    const int kvh = h0 / a.share;
    auto tile = [&](int key0) -> const char * {
        const int entry = entries[key0 >> a.page_shift];
        if ((unsigned)entry >= (uint64_t)a.n_pages) return nullptr;
        return a.v + ((((int64_t)entry * a.kv_heads + kvh) << a.page_shift) + (key0 & ((1 << a.page_shift) - 1))) * (D * (int)sizeof(T));
    };
    const float *const src = POST ? m.p1 : m.w_pre ? m.s2 : m.s1;       // (one row per head either way)
    value_rows<T, D, NT, GW> val;
    val.clear();
    for (int kb = beg; kb < end; kb += CH) {
        const int first = kb + wave * 16 * NT, key = first + mine;
        val.load(first, s.lo, end, lane, tile);
        const bool seen = key >= s.lo && key < end;
        const int at = seen ? key - s.base : 0;
#pragma unroll
        for (int g = 0; g < GW; ++g) {
            const float *x = src + ((int64_t)b * H + (h0 + g) / grp * grp) * m.span + at;
            float p = 0.0f;
#pragma unroll 4
            for (int i = sub; i < grp; i += SUBS) {
                const float2 c = coef[g * grp + i];
                const float v = x[(int64_t)i * m.span];
                p = fmaf(c.y, POST ? v : __builtin_amdgcn_exp2f(v * LOG2E - c.x), p);
            }
            if constexpr (SUBS >= 2) p = across32(p, [](float u, float v) { return u + v; });
            if constexpr (SUBS == 4) p = across16(p, [](float u, float v) { return u + v; });
            if (sub == 0) probs[g * 16 * NT + mine] = seen ? p : 0.0f;
        }
        wave_sync();
        val.multiply(probs, lane);
        wave_sync();
    }
    val.store(res + wave * GW * D, lane);
    __syncthreads();
    for (int x = tid; x < GW * D; x += 256) {
        float o = 0.0f;
#pragma unroll
        for (int w = 0; w < DECODE_WAVES; ++w) o += res[w * GW * D + x];
        if (m.v_splits == 1) out[x] = from_float<T>(o);
        else m.part[(((int64_t)b * H + h0 + x / D) * m.v_splits + split) * D + x % D] = o;
    }
}

template <typename T, int D> __global__ __launch_bounds__(256) void decode_sum_kernel(const mta_args m)
{
    constexpr int PARTS = 256 / D;
    __shared__ float so[PARTS][D];
    const int h = blockIdx.x, b = blockIdx.y, d = threadIdx.x % D, part = threadIdx.x / D;
    T *const out = (T *)m.d.o + ((int64_t)b * m.d.heads + h) * D;
    const slot_step s = step_of(m, b);
    if (s.n <= 0) {
        if (part == 0) out[d] = from_float<T>(s.n < 0 ? __builtin_nanf("") : 0.0f);
        return;
    }
    const int splits = (s.n - (s.lo & ~15) + m.v_len - 1) / m.v_len;
    const float *o = m.part + ((int64_t)b * m.d.heads + h) * m.v_splits * D + d;
    float sum = 0.0f;
#pragma unroll 8
    for (int i = part; i < splits; i += PARTS) sum += o[(int64_t)i * D];
    so[part][d] = sum;
    __syncthreads();
    if (part != 0) return;
#pragma unroll
    for (int i = 1; i < PARTS; ++i) sum += so[i][d];
    out[d] = from_float<T>(sum);
}

// ---- host side ----
struct plan {
    int nt, gw, split_len, n_splits, lds;             // scores
    int span, chunk, chunks;                          // mixing
    int v_nt, v_gw, v_len, v_splits, v_lds, mix_lds, post_lds;
    int64_t s1, s2, stats, p1, part, total;           // workspace, in floats
};

// keys per step (a power-of-two choice of `wide` and 1), and per split, for `groups` workgroups per split
void cut(int64_t span, int64_t groups, int wide, int &nt, int &len, int &splits)
{
    nt = (span + 64 * wide - 1) / (64 * wide) * groups >= 512 ? wide : 1;
    const int64_t steps = (span + 64 * nt - 1) / (64 * nt), per = (steps * groups + 1023) / 1024;
    len = (int)(per < steps ? per : steps) * 64 * nt;
    splits = (int)((span + len - 1) / len);
}

int plan_of(const mta_cache *c, int64_t longest, int R, int S, int R2, int S2, bool pre, bool post_conv, int pre_group, int post_group, int window, plan &p)
{
    const int size = dtype_size(c->dtype), share = c->heads / c->kv_heads, wide = c->head_dim * size > 256 ? 2 : 4, D = c->head_dim, W = R + R2 - 1;
    const int64_t span = span_of(longest, window, R2), H = c->heads, B = c->slots;
    p.gw = 0;
    for (int gw = 4; gw >= 1 && !p.gw; gw >>= 1) {
        if (share % gw) continue;
        cut(span, B * (H / gw), wide, p.nt, p.split_len, p.n_splits);
        p.lds = raw_layout_of(gw * W, R, S, gw, D, size, p.nt, false).total;
        if (p.nt > 1 && p.lds > 80 << 10) {
            cut(span, B * (H / gw), 1, p.nt, p.split_len, p.n_splits);
            p.lds = raw_layout_of(gw * W, R, S, gw, D, size, p.nt, false).total;
        }
        if (p.lds <= (gw == 1 ? 160 << 10 : 80 << 10)) p.gw = gw;
    }
    if (!p.gw) return MTA_ERR_KERNEL_SIZE;
    p.span = p.split_len * p.n_splits;
    // statistics: few chunks where many rows have to be put together from them
    const int most = R2 >= 8 ? 16 : 128 / R2;
    const int64_t tiles = (p.span + 63) / 64;
    p.chunk = (int)((tiles + most - 1) / most) * 64;
    p.chunks = (p.span + p.chunk - 1) / p.chunk;
    p.mix_lds = DECODE_WAVES * pre_group * 16;
    p.post_lds = (2 * R2 + R2 * S2 + R2 * (256 + S2 - 1)) * 4;
    p.v_gw = share % 4 == 0 ? 4 : share % 2 == 0 ? 2 : 1;
    cut(span_of(longest, window, 1), B * (H / p.v_gw), wide, p.v_nt, p.v_len, p.v_splits);
    p.v_lds = (2 * p.v_gw * post_group + DECODE_WAVES * p.v_gw * (16 * p.v_nt + D)) * 4;
    if (p.mix_lds > 160 << 10 || p.post_lds > 160 << 10 || p.v_lds > 160 << 10) return MTA_ERR_KERNEL_SIZE;
    p.s1 = 0;
    p.s2 = p.s1 + B * H * R2 * p.span;
    p.stats = p.s2 + (pre ? B * H * R2 * p.span : 0);
    p.p1 = p.stats + 2 * B * H * R2 * p.chunks;
    p.part = p.p1 + (post_conv ? B * H * p.span : 0);
    p.total = p.part + (p.v_splits > 1 ? B * H * p.v_splits * D : 0);
    return MTA_OK;
}

template <typename T, int D, int NT, int JB, bool ONE> int launch_scores(const mta_args &m, const plan &p, hipStream_t st)
{
    auto kern = decode_scores_kernel<T, D, NT, JB, ONE>;
    if (const int e = allow_lds(kern, p.lds)) return e;
    hipLaunchKernelGGL(kern, dim3((unsigned)p.n_splits, (unsigned)(m.d.heads / p.gw), (unsigned)m.d.slots), dim3(256), p.lds, st, m);
    return launch_status();
}
template <typename T, int D, int NT, int GW, bool POST> int launch_values(const mta_args &m, const plan &p, hipStream_t st)
{
    auto kern = decode_values_kernel<T, D, NT, GW, POST>;
    if (const int e = allow_lds(kern, p.v_lds)) return e;
    hipLaunchKernelGGL(kern, dim3((unsigned)p.v_splits, (unsigned)(m.d.heads / GW), (unsigned)m.d.slots), dim3(256), p.v_lds, st, m);
    return launch_status();
}
template <typename T, int D, int NT, bool POST> int launch_values_heads(const mta_args &m, const plan &p, hipStream_t st)
{
    return p.v_gw == 4 ? launch_values<T, D, NT, 4, POST>(m, p, st) : p.v_gw == 2 ? launch_values<T, D, NT, 2, POST>(m, p, st)
                                                                                   : launch_values<T, D, NT, 1, POST>(m, p, st);
}
template <typename T, int D, int NT> int launch_scores_rows(const mta_args &m, const plan &p, hipStream_t st)
{
    constexpr int SUBS = 16 / NT;
    return m.R2 == 1 ? launch_scores<T, D, NT, 1, true>(m, p, st) : m.R2 <= SUBS ? launch_scores<T, D, NT, 1, false>(m, p, st)
         : m.R2 <= 2 * SUBS ? launch_scores<T, D, NT, 2, false>(m, p, st) : launch_scores<T, D, NT, 3, false>(m, p, st);
}
template <typename T, int D> int launch_all(const mta_args &m, const plan &p, hipStream_t st)
{
    constexpr int WIDE = D * (int)sizeof(T) > 256 ? 2 : 4;
    const unsigned slots = (unsigned)m.d.slots, heads = (unsigned)m.d.heads;
    int e = p.nt == 1 ? launch_scores_rows<T, D, 1>(m, p, st) : launch_scores_rows<T, D, WIDE>(m, p, st);
    if (e) return e;
    if ((e = allow_lds(decode_mix_kernel, p.mix_lds))) return e;
    hipLaunchKernelGGL(decode_mix_kernel, dim3((unsigned)p.chunks, (unsigned)m.R2, slots), dim3(256), p.mix_lds, st, m);
    if (m.w2) {
        if ((e = allow_lds(decode_post_kernel, p.post_lds))) return e;
        hipLaunchKernelGGL(decode_post_kernel, dim3((unsigned)((p.span + 255) / 256), heads, slots), dim3(256), p.post_lds, st, m);
        e = p.v_nt == 1 ? launch_values_heads<T, D, 1, true>(m, p, st) : launch_values_heads<T, D, WIDE, true>(m, p, st);
    } else {
        e = p.v_nt == 1 ? launch_values_heads<T, D, 1, false>(m, p, st) : launch_values_heads<T, D, WIDE, false>(m, p, st);
    }
    if (e) return e;
    if (p.v_splits > 1) hipLaunchKernelGGL((decode_sum_kernel<T, D>), dim3(heads, slots), dim3(256), 0, st, m);
    return launch_status();
}

int check_args(const mta_cache *c, int64_t longest, int R, int S, int R2, int S2, int pre_group, int post_group, int window)
{
    if (const int e = check_cache(c)) return e;
    if (R < 1 || S < 1 || R2 < 1 || S2 < 1 || R > MTA_MAX_FUSED_KERNEL_R || S > MTA_MAX_FUSED_KERNEL_S || R2 > MTA_MAX_FUSED_KERNEL_R
        || S2 > MTA_MAX_FUSED_KERNEL_S)
        return MTA_ERR_KERNEL_SIZE;
    if (longest < 1 || longest > (int64_t)c->max_pages * c->page || window < 0 || c->query_rows < R + R2 - 1) return MTA_ERR_SHAPE;
    if (pre_group < 0 || post_group < 0 || (pre_group && c->heads % pre_group) || (post_group && c->heads % post_group)) return MTA_ERR_GROUP;
    return MTA_OK;
}

}  // namespace
}  // namespace mta

using namespace mta;

extern "C" int64_t mta_decode_workspace(const mta_cache *c, int64_t longest, int R, int S, int R2, int S2, int pre_group, int post_group, int window)
{
    if (const int e = check_args(c, longest, R, S, R2, S2, pre_group, post_group, window)) return e;
    plan p;
    // (the most that any choice of absent weights needs)
    if (const int e = plan_of(c, longest, R, S, R2, S2, true, true, pre_group ? pre_group : c->heads, post_group ? post_group : c->heads, window, p)) return e;
    return p.total * 4;
}

extern "C" int mta_decode(const mta_cache *c, const void *w, const void *w_pre, const void *w2, const void *w_post, void *o, void *workspace,
                          int64_t workspace_bytes, int64_t longest, int R, int S, int R2, int S2, int pre_group, int post_group, int window, float scale,
                          int w_dtype, void *stream)
{
    if (const int e = check_args(c, longest, R, S, R2, S2, pre_group, post_group, window)) return e;
    if (!w || !o || !workspace || (!w2 && (R2 != 1 || S2 != 1))) return MTA_ERR_NULL;
    const int ws = dtype_size(w_dtype);
    if (ws == 0) return MTA_ERR_DTYPE;
    if (!aligned_to(w, ws) || !aligned_to(w_pre, ws) || !aligned_to(w2, ws) || !aligned_to(w_post, ws) || !aligned_to(o, dtype_size(c->dtype)) || !aligned_to(workspace, 16))
        return MTA_ERR_ALIGN;
    mta_args m = {};
    m.pre_group = !w_pre ? 1 : pre_group ? pre_group : c->heads;
    m.post_group = !w_post ? 1 : post_group ? post_group : c->heads;
    plan p;
    if (const int e = plan_of(c, longest, R, S, R2, S2, w_pre != nullptr, w2 != nullptr, m.pre_group, m.post_group, window, p)) return e;
    if (workspace_bytes < p.total * 4) return MTA_ERR_WORKSPACE;
    m.d = args_of(c, w, R, S, R2, window, longest, scale, w_dtype);
    m.d.o = o, m.d.split_len = p.split_len, m.d.n_splits = p.n_splits, m.d.gw = p.gw;
    m.w_pre = w_pre, m.w_post = w_post, m.w2 = w2, m.R2 = R2, m.S2 = S2;
    m.span = p.span, m.chunk = p.chunk, m.chunks = p.chunks, m.v_len = p.v_len, m.v_splits = p.v_splits;
    float *const base = (float *)workspace;
    m.s1 = base + p.s1, m.s2 = base + p.s2, m.stats = base + p.stats, m.p1 = base + p.p1, m.part = base + p.part;
    const hipStream_t st = (hipStream_t)stream;
    MTA_DISPATCH_IO(c->dtype, return c->head_dim == 64 ? launch_all<io_t, 64>(m, p, st) : launch_all<io_t, 128>(m, p, st));
}
