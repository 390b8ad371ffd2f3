// Multi-Token Attention of the newest token of each slot of a paged cache.  With P the newest position, R x S and R2 x S2 the two conv
// kernels, and rows j = P - R2 + 1 .. P (the only ones that reach the newest row through the second conv):
//   raw_i[k] = scale * q_i . K_k where row i sees key k, else 0                       i = P - R2 - R + 2 .. P
//   s1_j[k]  = sum_{r, t} w[h][r][t] raw_{j - R + 1 + r}[k + t - (S-1)/2]              per head h
//   s2_j     = sum_g Wpre[h][g] s1_j (head g)                                         p_j = softmax over the keys that row j sees
//   p1[k]    = sum_{r, t} w2[h][r][t] p_{P - R2 + 1 + r}[k + t - (S2-1)/2]             p2 = sum_g Wpost[h][g] p1 (head g)
//   o        = sum_k p2[k] V_k
// Heads and rows meet between the stages, so this is not one pass but up to five kernels, two of which stream: scores (K once), mixing with the
// rows' statistics, the second conv (none where it is the identity: a single row is left then; one kernel with the mixing for short rows), mixing
// and values (V once), and the sum over the items.  What goes between them is R2 numbers of fp32 per key and head, against 2 D of K and V.
#include "decode.hpp"

namespace mta {
namespace {

struct mta_args {
    decode_args d;
    const void *w_pre, *w_post, *w2;
    int pre_group, post_group;  // heads that mix (1: the identity, no weight)
    int R2, S2, span;           // span: keys that a row of the workspace has room for
    int chunk, chunks;          // keys per workgroup of the mixing kernel
    int v_target, v_least, v_items, v_shift;   // the values kernel's items
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
    constexpr int CH = 64 * NT, SUBS = 16 / NT;
    const int lane = threadIdx.x & 63, groups = a.heads / a.gw, index = blockIdx.x / groups, h0 = (blockIdx.x - index * groups) * a.gw;
    const shares sh(a, m.R2 - 1, log2_of(CH), false, lane);
    const work_item it = item_of(sh, index, -1, lane);
    if (it.slot < 0 || it.s.n <= 0) return;
    const slot_step s = it.s;
    const int b = it.slot, beg = s.base + (index - it.first) * sh.per * CH, end = beg + sh.per * CH < s.n ? beg + sh.per * CH : s.n;
    page_map pages;
    pages.load(a, b, beg - halo_left(a.S), lane);

    using lanes = score_lanes<NT, 1>;
    const int rows = a.gw * a.W, right = a.S - 1 - (a.S - 1) / 2;
    const raw_layout l = raw_layout_of(rows, a.R, a.S, a.gw, D, (int)sizeof(T), NT, false);
    raw_scores<T, D, NT> sc(a, smem, l, pages, rows, h0 / a.share, s.n, end + right < s.n ? end + right : s.n);
    const int wave = sc.wave;
    const lanes me(lane);
    const float *const weights = reinterpret_cast<const float *>(smem + l.weights);
    const int sp = (a.S + 3) & ~3;

    typename raw_scores<T, D, NT>::start st;
    sc.begin(st, beg, b, h0);
    sc.load_step(beg);
    sc.finish(st, beg, b, h0, smem, l);
    int step = 0;
    for (int kb = beg; kb < end; kb += CH, ++step) {
        sc.score_step(kb, step);
        if (kb + CH < end) {   // (nothing else is under way here)
            sc.pages.reach(a, b, kb + CH, kb + 2 * CH + sc.hr < sc.limit ? kb + 2 * CH + sc.hr : sc.limit, lane);
            sc.load_step(kb + CH);
        }
        __syncthreads();
        const int local = wave * 16 * NT + 4 * me.quad, key = kb + local;
        float *const out = m.s1 + ((int64_t)b * a.heads + h0) * m.R2 * m.span + (key - s.base);
        for (int g = 0; g < a.gw; ++g) {
            const float *const w = weights + g * a.R * sp;
            if constexpr (ONE) {
                float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                with_taps(a.S, [&](auto count) {
                    for (int r = me.part; r < a.R; r += SUBS)
                        taps4<decltype(count)::value>(c, sc.window(step, g * a.W + r, local), w + r * sp, a.S);
                });
                me.deal(c);
                if (me.owner && key + lane / 16 < end) out[(int64_t)g * m.span + lane / 16] = c[0] * a.scale;
            } else {
                for (int j0 = me.part * JB; j0 < m.R2; j0 += SUBS * JB) {
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
// A wavefront takes blocks of four heads of a group, a lane four keys of each 256 (16 bytes per load); (reference, sum) run along per lane and meet
// at the end.
__global__ __launch_bounds__(256) void decode_mix_kernel(const mta_args m)
{
    extern __shared__ __align__(16) float lds[];
    const int b = blockIdx.z, j = blockIdx.x, chunk = blockIdx.y, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const slot_step s = step_of(m, b);
    if (s.n <= 0) return;
    const int k0 = s.base + chunk * m.chunk, pos = row_pos(m, s.n, j), H = m.d.heads, grp = m.pre_group;
    if (k0 >= s.n) return;
    const int end = k0 + m.chunk < s.n ? k0 + m.chunk : s.n, per = (grp + 3) / 4, blocks = H / grp * per;
    const int64_t head = (int64_t)m.R2 * m.span, row0 = (int64_t)b * H * head + (int64_t)j * m.span - s.base;
    f32x4 *const w = reinterpret_cast<f32x4 *>(lds) + wave * grp;
    for (int blk = wave; blk < blocks; blk += 4) {
        const int g0 = blk / per * grp, o0 = g0 + (blk % per) * 4, cnt = g0 + grp - o0 < 4 ? g0 + grp - o0 : 4;
        constexpr int AHEAD = 8;
        f32x4 first[AHEAD];   // (the first keys of the first heads: under way before the weights are)
        {
            const float *x = m.s1 + row0 + g0 * head + (k0 + 4 * lane < end ? k0 + 4 * lane : k0);
#pragma unroll
            for (int g = 0; g < AHEAD; ++g) first[g] = *reinterpret_cast<const f32x4 *>(x + (g < grp ? g : 0) * head);
        }
        if (m.w_pre) {
            wave_sync();
            for (int x = lane; x < grp * 4; x += 64)
                lds[wave * grp * 4 + x] = (x & 3) < cnt ? load_any(m.w_pre, m.d.w_dtype, (int64_t)(o0 + (x & 3)) * H + g0 + (x >> 2)) : 0.0f;
            wave_sync();
        }
        float top[4], sum[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) top[u] = -INFINITY, sum[u] = 0.0f;
        for (int key = k0 + 4 * lane; key < end; key += 256) {   // (a row has room for whole vectors)
            f32x4 c[4];
            const float *x = m.s1 + row0 + g0 * head + key;
            const bool begun = key < k0 + 256;
            if (m.w_pre) {
#pragma unroll
                for (int u = 0; u < 4; ++u) c[u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                auto add = [&](int g, const f32x4 &v) {
                    const f32x4 wg = w[g];
#pragma unroll
                    for (int u = 0; u < 4; ++u)
#pragma unroll
                        for (int e = 0; e < 4; ++e) c[u][e] = fmaf(wg[u], v[e], c[u][e]);
                };
                if (begun) {
#pragma unroll
                    for (int g = 0; g < AHEAD; ++g)
                        if (g < grp) add(g, first[g]);
                }
#pragma unroll 8
                for (int g = begun ? AHEAD : 0; g < grp; ++g) add(g, *reinterpret_cast<const f32x4 *>(x + g * head));
            } else {
                c[0] = begun ? first[0] : *reinterpret_cast<const f32x4 *>(x);   // (groups of one head)
                c[1] = c[2] = c[3] = c[0];
            }
            bool seen[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) seen[e] = key + e < end && sees(m, pos, key + e);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (m.w_pre && u < cnt) *reinterpret_cast<f32x4 *>(m.s2 + row0 + (o0 + u) * head + key) = c[u];
                float t = top[u];
#pragma unroll
                for (int e = 0; e < 4; ++e) t = fmaxf(t, seen[e] ? c[u][e] * LOG2E : -INFINITY);
                const float ref = t == -INFINITY ? 0.0f : t;
                sum[u] *= __builtin_amdgcn_exp2f(top[u] - ref);
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[u] += seen[e] ? __builtin_amdgcn_exp2f(fmaf(c[u][e], LOG2E, -ref)) : 0.0f;
                top[u] = t;
            }
        }
        // (all four heads, whether they are there or not: their reductions run beside one another)
        float t[4], l[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) t[u] = wave_max(top[u]);
#pragma unroll
        for (int u = 0; u < 4; ++u) l[u] = wave_sum(sum[u] * __builtin_amdgcn_exp2f(top[u] - (t[u] == -INFINITY ? 0.0f : t[u])));
        if (lane < cnt) {
            const float tl = lane == 0 ? t[0] : lane == 1 ? t[1] : lane == 2 ? t[2] : t[3], ll = lane == 0 ? l[0] : lane == 1 ? l[1] : lane == 2 ? l[2] : l[3];
            *reinterpret_cast<float2 *>(m.stats + ((((int64_t)b * H + o0 + lane) * m.R2 + j) * m.chunks + chunk) * 2) = make_float2(tl, ll);
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
// A wavefront takes 256 keys of one head, four to a lane: those that its taps reach included, so that a row is one load.  Its probabilities lie in
// its own part of LDS.
__host__ __device__ __forceinline__ int post_left(int S2) { return ((S2 - 1) / 2 + 3) & ~3; }
__host__ __device__ __forceinline__ int post_keys(int S2) { return 256 - post_left(S2) - ((S2 - 1 - (S2 - 1) / 2 + 3) & ~3); }   // results
__host__ __device__ __forceinline__ int post_blocks(int span, int S2) { return (span + post_keys(S2) - 1) / post_keys(S2); }
constexpr int POST_STRIDE = 256 + 12;
__host__ __device__ __forceinline__ int post_floats(int R2, int S2) { return 2 * up16(R2) + R2 * (((S2 + 3) & ~3) + POST_STRIDE); }

// SPLIT: the four wavefronts of a workgroup take the same keys of one head and deal its rows out among them, which shortens the chain of a wavefront
// and costs four times the starts and a sum: for more than eight rows, and for fewer while the workgroups are no more than 192 to a row.  All kernels
// of a call, us, split | not (slots x heads, keys, R2 x S2): 1 x 8, 1500: 3 x 3 21.6 | 22.6, 11 x 15 22.4 | 27.7; 16 x 16, 600 (768 workgroups):
// 3 x 3 33.9 | 33.8, 6 x 9 30.8 | 31.6, 11 x 15 33.2 | 37.2; 16 x 16, 4000 (4352): 3 x 3 86.7 | 82.2, 6 x 9 95.8 | 94.0, 11 x 15 111.7 | 117.4.
template <bool SPLIT> __global__ __launch_bounds__(256) void decode_post_kernel(const mta_args m)
{
    extern __shared__ __align__(16) float lds[];
    const int b = blockIdx.z, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), H = m.d.heads;
    const int h = SPLIT ? blockIdx.x : blockIdx.x * (blockDim.x >> 6) + wave;
    const slot_step s = step_of(m, b);
    const int k0 = s.base + blockIdx.y * post_keys(m.S2);
    if (h >= H || s.n <= 0 || k0 >= s.n) return;   // (SPLIT: all four wavefronts or none; else nothing below waits for another one)
    const int r0 = SPLIT ? wave * m.R2 / 4 : 0, R2 = (SPLIT ? (wave + 1) * m.R2 / 4 : m.R2) - r0;   // rows
    const int left = (m.S2 - 1) / 2, left4 = post_left(m.S2), shift = left & 3, taps = R2 * m.S2, sp = (m.S2 + 3) & ~3;
    float *const mine = lds + wave * post_floats(SPLIT ? (m.R2 + 3) / 4 : R2, m.S2), *const w = mine + 2 * up16(R2), *const p = w + R2 * sp;
    float2 *const stat = reinterpret_cast<float2 *>(mine);
    const int64_t row0 = ((int64_t)b * H + h) * m.R2 + r0;
    const int chunks = (s.n - s.base + m.chunk - 1) / m.chunk;
    // (loads first: scores, which do not wait for the statistics, then weights and statistics)
    constexpr int AHEAD = SPLIT ? 4 : 8;
    const int key0 = k0 - left4 + 4 * lane;
    const float *const sc = (m.w_pre ? m.s2 : m.s1) + row0 * m.span + (key0 >= s.base && key0 < s.n ? key0 - s.base : 0);
    f32x4 x[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) x[j] = *reinterpret_cast<const f32x4 *>(sc + (int64_t)(j < R2 ? j : 0) * m.span);
#pragma unroll 4
    for (int t = lane; t < taps; t += 64) w[t / m.S2 * sp + t % m.S2] = load_any(m.w2, m.d.w_dtype, ((int64_t)h * m.R2 + r0) * m.S2 + t);
    for (int t = lane; t < R2 * 8; t += 64) {
        const float2 st = row_statistics<8>(m.stats + (row0 + t / 8) * m.chunks * 2, chunks, t % 8);
        if (t % 8 == 0) stat[t / 8] = st;
    }
    wave_sync();
    for (int j0 = 0; j0 < R2; j0 += AHEAD) {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            if (j0 + j >= R2) break;
            const int pos = row_pos(m, s.n, r0 + j0 + j);
            const float2 st = stat[j0 + j];
            float *const to = p + (j0 + j) * POST_STRIDE + shift + 4 * lane;   // (the taps of a lane's keys begin on 16 bytes)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                to[e] = key0 + e >= s.base && sees(m, pos, key0 + e) ? __builtin_amdgcn_exp2f(fmaf(x[j][e], LOG2E, -st.x)) * st.y : 0.0f;
        }
        if (j0 + AHEAD < R2) {
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) x[j] = *reinterpret_cast<const f32x4 *>(sc + (int64_t)(j0 + AHEAD + j < R2 ? j0 + AHEAD + j : 0) * m.span);
        }
    }
    wave_sync();
    const int key = k0 + 4 * lane;
    const bool there = 4 * lane < post_keys(m.S2) && key < s.n;
    if (!SPLIT && !there) return;
    float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const float *const from = p + shift + 4 * lane + left4 - left;
    if (there)
        with_taps(m.S2, [&](auto count) {
            for (int j = 0; j < R2; ++j) taps4<decltype(count)::value>(c, from + j * POST_STRIDE, w + j * sp, m.S2);
        });
    if constexpr (SPLIT) {
        __syncthreads();
        *reinterpret_cast<f32x4 *>(lds + 256 * wave + 4 * lane) = f32x4{c[0], c[1], c[2], c[3]};
        __syncthreads();
        if (wave || !there) return;
#pragma unroll
        for (int o = 1; o < 4; ++o)
#pragma unroll
            for (int e = 0; e < 4; ++e) c[e] += lds[256 * o + 4 * lane + e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) c[e] = key + e >= s.lo ? c[e] : 0.0f;
    *reinterpret_cast<f32x4 *>(m.p1 + ((int64_t)b * H + h) * m.span + (key - s.base)) = f32x4{c[0], c[1], c[2], c[3]};
}

// ---- mixing, softmax and the conv behind it in one kernel, for rows of up to 512 keys ----
// A workgroup takes a block of up to four heads of a group; a wavefront an output row of all four, whole, 4 KQ keys to a lane, so that neither the
// mixed scores nor statistics go through memory; then a wavefront 256 keys of one head for the conv, from the probabilities in LDS.  Eight
// wavefronts, 16 above eight rows: a row more to a wavefront is a turn of loads more (rows 5 to 8 with four wavefronts: 3 us slower).
// All kernels of a call, us, one kernel | two (3 x 3 in front; slots x heads, R2 x S2, heads that mix):
//   250 keys  1 x 8, 3 x 3, all 16.1 | 19.3    2 x 16, 10 x 11, 4 19.1 | 26.4    32 x 16, 7 x 7, all 29.8 | 35.3
//   500 keys  1 x 8, 3 x 3, all 18.4 | 20.6    2 x 16, 10 x 11, 4 21.9 | 27.9    32 x 16, 7 x 7, all 43.9 | 49.1
// and with 16 keys to a lane, 1000 keys 22.3 | 21.7, 28.5 | 28.3, 78.3 | 80.5: the chain in a wavefront grows while the two kernels spread, so
// longer rows stay with those.
__host__ __device__ __forceinline__ int short_stride(int S2, int kq) { return post_left(S2) + 256 * kq + 12 + up16(S2); }
__host__ __device__ __forceinline__ int short_floats(int R2, int S2, int pre_group, int kq)
{
    return 4 * pre_group + 4 * R2 * ((S2 + 3) & ~3) + 4 * R2 * short_stride(S2, kq);
}

template <int KQ> __global__ __launch_bounds__(1024) void decode_mix_post_kernel(const mta_args m)
{
    extern __shared__ __align__(16) float lds[];
    const int tid = threadIdx.x, threads = blockDim.x, waves = threads >> 6, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int b = blockIdx.y, H = m.d.heads, R2 = m.R2, S2 = m.S2;
    const slot_step s = step_of(m, b);
    if (s.n <= 0) return;
    const int grp = m.pre_group, per = (grp + 3) / 4, blk = blockIdx.x, g0 = blk / per * grp, o0 = g0 + blk % per * 4;
    const int cnt = g0 + grp - o0 < 4 ? g0 + grp - o0 : 4, keys = s.n - s.base, taps = R2 * S2;
    const int left = (S2 - 1) / 2, left4 = post_left(S2), shift = left & 3, stride = short_stride(S2, KQ), sp = (S2 + 3) & ~3;
    // (rows: a row's key 0; the taps of every fourth key begin on 16 bytes)
    float *const w = lds, *const w2 = w + 4 * grp, *const rows = w2 + 4 * R2 * sp + left4 + shift;
    const int64_t head = (int64_t)R2 * m.span;
    if (m.w_pre)
        for (int x = tid; x < grp * 4; x += threads) w[x] = (x & 3) < cnt ? load_any(m.w_pre, m.d.w_dtype, (int64_t)(o0 + (x & 3)) * H + g0 + (x >> 2)) : 0.0f;
#pragma unroll 2
    for (int x = tid; x < cnt * taps; x += threads) w2[x / S2 * sp + x % S2] = load_any(m.w2, m.d.w_dtype, (int64_t)o0 * taps + x);
    for (int r = wave; r < 4 * R2; r += waves) {   // zeros on either side of every row's keys
        float *const row = rows + r * stride;
        if (lane < left4 + shift) row[lane - left4 - shift] = 0.0f;
        for (int c = keys + lane; c < stride - left4 - shift; c += 64) row[c] = 0.0f;
    }
    __syncthreads();
    for (int j = wave; j < R2; j += waves) {
        const float *const x = m.s1 + ((int64_t)b * H + g0) * head + (int64_t)j * m.span;
        const int pos = row_pos(m, s.n, j);
        f32x4 c[4][KQ];
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int q = 0; q < KQ; ++q) c[u][q] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
        for (int g = 0; g < grp; ++g) {
            const f32x4 wg = m.w_pre ? *reinterpret_cast<const f32x4 *>(w + 4 * g) : f32x4{1.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int q = 0; q < KQ; ++q) {
                const int k = 256 * q + 4 * lane;
                const f32x4 v = *reinterpret_cast<const f32x4 *>(x + g * head + (k < keys ? k : 0));   // (a row has room for whole vectors)
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int e = 0; e < 4; ++e) c[u][q][e] = fmaf(wg[u], v[e], c[u][q][e]);
            }
        }
        float top[4], sum[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            top[u] = -INFINITY;
#pragma unroll
            for (int q = 0; q < KQ; ++q)
#pragma unroll
                for (int e = 0; e < 4; ++e) top[u] = fmaxf(top[u], sees(m, pos, s.base + 256 * q + 4 * lane + e) ? c[u][q][e] * LOG2E : -INFINITY);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) top[u] = wave_max(top[u]);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const float ref = top[u] == -INFINITY ? 0.0f : top[u];
            sum[u] = 0.0f;
#pragma unroll
            for (int q = 0; q < KQ; ++q)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    c[u][q][e] = sees(m, pos, s.base + 256 * q + 4 * lane + e) ? __builtin_amdgcn_exp2f(fmaf(c[u][q][e], LOG2E, -ref)) : 0.0f;
                    sum[u] += c[u][q][e];
                }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) sum[u] = wave_sum(sum[u]);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (u >= cnt) break;
            const float f = pos >= 0 ? 1.0f / sum[u] : 0.0f;   // (a row ahead of the first token sees nothing)
            float *const to = rows + (u * R2 + j) * stride;
#pragma unroll
            for (int q = 0; q < KQ; ++q)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int k = 256 * q + 4 * lane + e;
                    if (k < keys) to[k] = c[u][q][e] * f;
                }
        }
    }
    __syncthreads();
    const int u = wave & 3;   // (eight or 16 wavefronts)
    if (u >= cnt) return;
    for (int k = 256 * (wave >> 2) + 4 * lane; k < keys; k += 64 * waves) {
        float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        with_taps(S2, [&](auto count) {
            for (int j = 0; j < R2; ++j) taps4<decltype(count)::value>(c, rows + (u * R2 + j) * stride + k - left, w2 + (u * R2 + j) * sp, S2);
        });
#pragma unroll
        for (int e = 0; e < 4; ++e) c[e] = s.base + k + e >= s.lo ? c[e] : 0.0f;
        *reinterpret_cast<f32x4 *>(m.p1 + ((int64_t)b * H + o0 + u) * m.span + k) = f32x4{c[0], c[1], c[2], c[3]};
    }
}

// ---- mixing behind the softmax and P V: V once ----
// POST: p1 has been through the second conv; else the heads' probabilities are formed here, from scores and statistics.
template <typename T, int D, int NT, int GW, bool POST>
__global__ __launch_bounds__(256) void decode_values_kernel(const mta_args m)
{
    extern __shared__ __align__(16) float lds[];
    decode_args a = m.d;
    a.target = m.v_target, a.least = m.v_least, a.items = m.v_items;
    constexpr int CH = 64 * NT;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), H = a.heads, grp = m.post_group;
    const int groups = H / GW, index = blockIdx.x / groups, h0 = (blockIdx.x - index * groups) * GW;
    const shares sh(a, m.R2 - 1, log2_of(CH), true, lane);
    const work_item it = item_of(sh, index, -1, lane);
    if (it.slot < 0) return;
    const slot_step s = it.s;
    const int b = it.slot;
    T *const out = (T *)a.o + ((int64_t)b * H + h0) * D;
    if (s.n <= 0) {
        for (int x = tid; x < GW * D; x += 256) out[x] = from_float<T>(s.n < 0 ? __builtin_nanf("") : 0.0f);
        return;
    }
    const int beg = (s.lo & ~15) + (index - it.first) * sh.per * CH, end = beg + sh.per * CH < s.n ? beg + sh.per * CH : s.n;
    page_map pages;
    pages.load(a, b, beg, lane);
    using lanes = score_lanes<NT, GW>;
    const lanes me(lane);
    float2 *const coef = reinterpret_cast<float2 *>(lds);               // [GW][grp]: reference, weight / sum
    float *const probs = lds + 2 * up16(GW * grp) + wave * GW * 16 * NT;
    float *const res = lds + 2 * up16(GW * grp) + DECODE_WAVES * GW * 16 * NT;
    const int kvh = h0 / a.share;

    // what a lane mixes: its quad's keys of the heads part, part + RG, .. of its head's group
    const float *const src = (POST ? m.p1 : m.w_pre ? m.s2 : m.s1) + ((int64_t)b * H + (h0 + me.head) / grp * grp) * m.span - s.base;   // (one row per head)
    const float2 *const mix = coef + me.head * grp;
    constexpr int AHEAD = 2;    // loads of the next step that are under way while this one is multiplied
    f32x4 next[AHEAD];
    value_rows<T, D, NT, GW> val;
    auto fetch = [&](int i, int first) {
        const int key = first + 4 * me.quad;   // (whole vectors: where the quad begins behind the last key, of the row's first ones)
        return *reinterpret_cast<const f32x4 *>(src + (int64_t)(i < grp ? i : 0) * m.span + (key < s.n ? key : s.base));
    };
    auto ahead = [&](int kb) {
        const int first = kb + wave * 16 * NT;
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) next[u] = fetch(me.part + u * lanes::RG, first);
        val.load(a, pages, kvh, first, s.lo, end, lane);
    };
    ahead(beg);
    val.clear();
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
    auto advance = [&](int kb, auto more) {
        const int first = kb + wave * 16 * NT;
        float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        auto add = [&](int i, const f32x4 &v) {
            if (i < grp) {
                const float2 f = mix[i];
#pragma unroll
                for (int e = 0; e < 4; ++e) c[e] = fmaf(f.y, POST ? v[e] : __builtin_amdgcn_exp2f(fmaf(v[e], LOG2E, -f.x)), c[e]);
            }
        };
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) add(me.part + u * lanes::RG, next[u]);
#pragma unroll 4
        for (int i = me.part + AHEAD * lanes::RG; i < grp; i += lanes::RG) add(i, fetch(i, first));
        me.deal(c);
        if (me.owner) {
#pragma unroll
            for (int u = 0; u < lanes::VALUES; ++u) {
                const int key = first + me.key + u;
                probs[me.head * 16 * NT + me.key + u] = key >= s.lo && key < end ? c[u] : 0.0f;
            }
        }
        wave_sync();
        val.multiply(probs, first, s.lo, end, lane);
        if constexpr (more.value) {
            pages.reach(a, b, kb + CH, kb + 2 * CH < end ? kb + 2 * CH : end, lane);
            ahead(kb + CH);
        }
        wave_sync();
    };
    int kb = beg;
    for (; kb + CH < end; kb += CH) advance(kb, count_of<1>());
    advance(kb, count_of<0>());
    val.store(res + wave * GW * D, lane);
    __syncthreads();
    for (int x = tid; x < GW * D; x += 256) {
        float o = 0.0f;
#pragma unroll
        for (int w = 0; w < DECODE_WAVES; ++w) o += res[w * GW * D + x];
        if (it.count == 1) out[x] = from_float<T>(o);
        else m.part[((int64_t)index * H + h0) * D + x] = o;
    }
}

template <typename T, int D> __global__ __launch_bounds__(256) void decode_sum_kernel(const mta_args m)
{
    constexpr int PARTS = 1024 / D;   // (four elements to a lane)
    __shared__ __align__(16) float so[PARTS][D];
    decode_args a = m.d;
    a.target = m.v_target, a.least = m.v_least, a.items = m.v_items;
    const int h = blockIdx.x, b = blockIdx.y, d = threadIdx.x % (D / 4) * 4, part = threadIdx.x / (D / 4), lane = threadIdx.x & 63;
    const shares sh(a, m.R2 - 1, m.v_shift, true, lane);
    const work_item it = item_of(sh, 0, b, lane);
    if (it.count == 1) return;   // (that item wrote the result)
    T *const out = (T *)a.o + ((int64_t)b * a.heads + h) * D;
    const float *o = m.part + ((int64_t)it.first * a.heads + h) * D + d;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int i = part; i < it.count; i += PARTS) sum += *reinterpret_cast<const f32x4 *>(o + (int64_t)i * a.heads * D);
    *reinterpret_cast<f32x4 *>(&so[part][d]) = sum;
    __syncthreads();
    if (threadIdx.x >= D) return;
    float all = 0.0f;
#pragma unroll
    for (int i = 0; i < PARTS; ++i) all += so[i][threadIdx.x];
    out[threadIdx.x] = from_float<T>(all);
}

// ---- host side ----
struct plan {
    cut t, v;                                         // items of the scores and of the values kernel
    int gw, lds;                                      // scores
    int span, chunk, chunks, v_gw, v_lds, mix_lds, post_waves, post_lds, post_split, short_kq, short_lds;   // short_kq: 256s of keys in a short row, or 0
    int64_t s1, s2, stats, p1, part, total;           // workspace, in floats
};

int plan_of(const mta_cache *c, int64_t longest, int R, int S, int R2, int S2, bool pre, bool post_conv, int pre_group, int post_group, int window, plan &p)
{
    const int size = dtype_size(c->dtype), share = c->heads / c->kv_heads, D = c->head_dim, W = R + R2 - 1;
    const int64_t span = span_of(longest, window, R2), H = c->heads, B = c->slots;
    for (p.gw = 4; p.gw >= 1; p.gw >>= 1) {
        if (share % p.gw) continue;
        int most = most_tiles(D * size);
        while (most > 1 && raw_layout_of(p.gw * W, R, S, p.gw, D, size, most, false).total > 80 << 10) most >>= 1;
        p.t = cut_of(span, B, H / p.gw, most, 1024, false);
        p.lds = raw_layout_of(p.gw * W, R, S, p.gw, D, size, p.t.nt, false).total;
        if (p.lds <= (p.gw == 1 ? 160 << 10 : 80 << 10)) break;
    }
    if (!p.gw) return MTA_ERR_KERNEL_SIZE;
    p.span = (int)((span + 255) / 256 * 256);
    // statistics: few chunks where many rows have to be put together from them
    const int most = R2 >= 8 ? 16 : 128 / R2, tiles = p.span / 256;
    p.chunk = (tiles + most - 1) / most * 256;
    p.chunks = (p.span + p.chunk - 1) / p.chunk;
    p.mix_lds = DECODE_WAVES * pre_group * 16;
    for (p.post_waves = 4; p.post_waves > 1 && p.post_waves * post_floats(R2, S2) * 4 > 64 << 10;) p.post_waves >>= 1;
    p.post_lds = p.post_waves * post_floats(R2, S2) * 4;
    p.post_split = R2 > 1 && (R2 > 8 || H * B * post_blocks(p.span, S2) <= 192 * R2);
    if (p.post_split) p.post_waves = 4, p.post_lds = 16 * post_floats((R2 + 3) / 4, S2);
    p.short_kq = !post_conv ? 0 : p.span == 256 ? 1 : p.span == 512 ? 2 : 0;
    p.short_lds = short_floats(R2, S2, pre_group, p.short_kq) * 4;
    if (p.short_lds > 160 << 10) p.short_kq = 0;
    p.v_gw = share % 4 == 0 ? 4 : share % 2 == 0 ? 2 : 1;
    p.v = cut_of(span_of(longest, window, 1), B, H / p.v_gw, most_tiles(D * size), 1024, true);
    p.v_lds = (2 * up16(p.v_gw * post_group) + DECODE_WAVES * p.v_gw * (16 * p.v.nt + D)) * 4;
    if (too_many(p.t, H / p.gw) || too_many(p.v, H / p.v_gw)) return MTA_ERR_SHAPE;
    if (p.mix_lds > 160 << 10 || p.v_lds > 160 << 10) return MTA_ERR_SHAPE;
    if (p.post_lds > 160 << 10) return MTA_ERR_KERNEL_SIZE;
    p.s1 = 0;
    p.s2 = p.s1 + B * H * R2 * p.span;
    p.stats = p.s2 + (pre ? B * H * R2 * p.span : 0);
    p.p1 = p.stats + (2 * B * H * R2 * p.chunks + 3) / 4 * 4;   // (parts begin on 16 bytes; the others are whole vectors as they are)
    p.part = p.p1 + (post_conv ? B * H * p.span : 0);
    p.total = p.part + (p.v.joined ? (int64_t)p.v.items * H * D : 0);
    return MTA_OK;
}

template <typename T, int D, int NT, int JB, bool ONE> int launch_scores(const mta_args &m, const plan &p, hipStream_t st)
{
    auto kern = decode_scores_kernel<T, D, NT, JB, ONE>;
    if (const int e = allow_lds(kern, p.lds)) return e;
    hipLaunchKernelGGL(kern, dim3((unsigned)(p.t.items * (m.d.heads / p.gw))), dim3(256), p.lds, st, m);
    return launch_status();
}
template <typename T, int D, int NT, int GW, bool POST> int launch_values(const mta_args &m, const plan &p, hipStream_t st)
{
    auto kern = decode_values_kernel<T, D, NT, GW, POST>;
    if (const int e = allow_lds(kern, p.v_lds)) return e;
    hipLaunchKernelGGL(kern, dim3((unsigned)(p.v.items * (m.d.heads / GW))), dim3(256), p.v_lds, st, m);
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
template <typename T, int D, int NT> int launch_values_conv(const mta_args &m, const plan &p, hipStream_t st)
{
    return m.w2 ? launch_values_heads<T, D, NT, true>(m, p, st) : launch_values_heads<T, D, NT, false>(m, p, st);
}
template <typename T, int D> int launch_all(const mta_args &m, const plan &p, hipStream_t st)
{
    constexpr int MOST = most_tiles(D * (int)sizeof(T));
    const unsigned slots = (unsigned)m.d.slots, heads = (unsigned)m.d.heads;
    int e = MTA_ERR_UNSUPPORTED;
    if (p.t.nt == 1) e = launch_scores_rows<T, D, 1>(m, p, st);
    if constexpr (MOST >= 2)
        if (p.t.nt == 2) e = launch_scores_rows<T, D, 2>(m, p, st);
    if constexpr (MOST >= 4)
        if (p.t.nt == 4) e = launch_scores_rows<T, D, 4>(m, p, st);
    if (e) return e;
    if (p.short_kq) {
        const dim3 grid(heads / m.pre_group * ((m.pre_group + 3) / 4), slots);
        auto kern = p.short_kq == 1 ? decode_mix_post_kernel<1> : decode_mix_post_kernel<2>;
        if ((e = allow_lds(kern, p.short_lds))) return e;
        hipLaunchKernelGGL(kern, grid, dim3(m.R2 <= 8 ? 512 : 1024), p.short_lds, st, m);
    } else {
        if ((e = allow_lds(decode_mix_kernel, p.mix_lds))) return e;
        hipLaunchKernelGGL(decode_mix_kernel, dim3((unsigned)m.R2, (unsigned)p.chunks, slots), dim3(256), p.mix_lds, st, m);
        if (m.w2) {
            auto kern = p.post_split ? decode_post_kernel<true> : decode_post_kernel<false>;
            if ((e = allow_lds(kern, p.post_lds))) return e;
            const int at_once = p.post_split ? 1 : p.post_waves;
            const dim3 grid((heads + at_once - 1) / at_once, (unsigned)post_blocks(p.span, m.S2), slots);
            hipLaunchKernelGGL(kern, grid, dim3(64 * p.post_waves), p.post_lds, st, m);
        }
    }
    e = MTA_ERR_UNSUPPORTED;
    if (p.v.nt == 1) e = launch_values_conv<T, D, 1>(m, p, st);
    if constexpr (MOST >= 2)
        if (p.v.nt == 2) e = launch_values_conv<T, D, 2>(m, p, st);
    if constexpr (MOST >= 4)
        if (p.v.nt == 4) e = launch_values_conv<T, D, 4>(m, p, st);
    if (e) return e;
    if (p.v.joined) hipLaunchKernelGGL((decode_sum_kernel<T, D>), dim3(heads, slots), dim3(256), 0, st, m);
    return launch_status();
}

int check_args(const mta_cache *c, int64_t longest, int R, int S, int R2, int S2, int pre_group, int post_group, int window)
{
    if (const int e = check_cache(c)) return e;
    if (R < 1 || S < 1 || R2 < 1 || S2 < 1 || R > MTA_MAX_FUSED_KERNEL_R || S > MTA_MAX_FUSED_KERNEL_S || R2 > MTA_MAX_FUSED_KERNEL_R
        || S2 > MTA_MAX_FUSED_KERNEL_S)
        return MTA_ERR_KERNEL_SIZE;
    if (longest < 1 || longest > MTA_MAX_DECODE_KEYS || longest > (int64_t)c->max_pages * c->page || window < 0 || c->query_rows < R + R2 - 1) return MTA_ERR_SHAPE;
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
    m.d.o = o, m.d.target = p.t.target, m.d.least = p.t.least, m.d.items = p.t.items, m.d.gw = p.gw;
    m.w_pre = w_pre, m.w_post = w_post, m.w2 = w2, m.R2 = R2, m.S2 = S2;
    m.span = p.span, m.chunk = p.chunk, m.chunks = p.chunks, m.v_target = p.v.target, m.v_least = p.v.least, m.v_items = p.v.items, m.v_shift = 6 + (p.v.nt >> 1);   // (nt: 1, 2 or 4)
    float *const base = (float *)workspace;
    m.s1 = base + p.s1, m.s2 = base + p.s2, m.stats = base + p.stats, m.p1 = base + p.p1, m.part = base + p.part;
    const hipStream_t st = (hipStream_t)stream;
    MTA_DISPATCH_IO(c->dtype, return c->head_dim == 64 ? launch_all<io_t, 64>(m, p, st) : launch_all<io_t, 128>(m, p, st));
}
