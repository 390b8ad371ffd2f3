// What the kernels of single-token attention over a paged cache share (decode_attn.hip, decode_mta.hip).
//
// A slot b holds n tokens: the ones it had (state[0][b]) and the ones it got last (state[1][b]; none: the slot sits this step out).  The newest
// query row is p = n - 1.  Keys and values lie in pages (page, key head, row, element), table[b][key / page] names the page; queries in a
// ring, position i in row i % ring.  A row i sees the keys max(0, i - window + 1) .. i; what a row does not see counts as 0 ahead of the conv.
//
// Work split.  A workgroup of four wavefronts takes one slot, one or more query heads of one key head, and a stretch of the keys (a "split"),
// in steps of 64 * NT keys, 16 * NT per wavefront.  Keys are a tile of 16 consecutive rows of a page, read straight into the operand
// fragments of 16x16 products (no key is used by two wavefronts, so LDS would only add a pass); the query rows that the conv needs, one to a
// few tens, are the other operand, in LDS.  The conv takes what it needs of neighbouring keys from LDS, where the last columns of a step are
// written a second time, as the first columns of the next one: a split reads (halo) keys twice only where it begins.  Three buffers of raw
// scores: one is read, the next one gets the columns to come, and the one before may still be read by a wavefront that is behind - a single
// barrier per step.
#pragma once

#include "common.hpp"
#include "mfma.hpp"

namespace mta {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
constexpr float LOG2E = 1.4426950408889634f;
constexpr int DECODE_WAVES = 4;

struct decode_args {
    const char *k, *v, *q;      // pools and ring
    const void *w;              // conv weights (H, R, S)
    const int *table, *state;
    float *ws;                  // partial results / scores
    void *o;
    int64_t n_pages;
    int slots, max_pages, page_shift, heads, kv_heads, share, ring;
    int R, S, W;                // conv kernel; query rows of raw scores (R + output rows - 1)
    int w_dtype, window, longest;
    int split_len, n_splits;    // keys per split; splits that the grid and the workspace have room for
    int gw;                     // query heads per workgroup
    float scale;
};

// One slot's step: n < 0: not a state of this cache, or more tokens than grid and workspace were sized for (its outputs are NaN); 0: it
// sits this step out (zeros).  older: output rows ahead of the newest one.
// base: where the splits begin, a multiple of 16; lo: the first key that the newest row sees.
struct slot_step { int n, base, lo; };
__device__ __forceinline__ slot_step step_of(const decode_args &a, int b, int older)
{
    const int had = a.state[b], got = a.state[a.slots + b];
    slot_step s = {0, 0, 0};
    if (got <= 0) return s;
    s.n = had + got;
    if (had < 0 || s.n <= 0 || s.n > a.longest) { s.n = -1; return s; }
    if (a.window > 0) {
        s.lo = s.n > a.window ? s.n - a.window : 0;
        s.base = s.lo > older ? (s.lo - older) & ~15 : 0;   // (the first key of the oldest output row)
    }
    return s;
}

// What one lane of a wavefront left in LDS is there for the others (LDS serves a wavefront in order; this holds the compiler to it).
__device__ __forceinline__ void wave_sync()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

// ---- reductions over a wavefront on the vector ALU: rows of 16 lanes by rotations, then across rows ----
template <int CTRL> __device__ __forceinline__ float dpp(float v)
{
    return __uint_as_float((unsigned)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, 0xf, 0xf, false));
}
template <typename F> __device__ __forceinline__ float across16(float v, F op)
{
    uint32_t a = __float_as_uint(v), b = a;
    swap16(a, b);
    return op(__uint_as_float(a), __uint_as_float(b));
}
template <typename F> __device__ __forceinline__ float across32(float v, F op)
{
    uint32_t a = __float_as_uint(v), b = a;
    swap32(a, b);
    return op(__uint_as_float(a), __uint_as_float(b));
}
template <typename F> __device__ __forceinline__ float wave_reduce(float v, F op)
{
    v = op(v, dpp<0x128>(v));
    v = op(v, dpp<0x124>(v));
    v = op(v, dpp<0x122>(v));
    v = op(v, dpp<0x121>(v));
    return across32(across16(v, op), op);
}
__device__ __forceinline__ float wave_max(float v) { return wave_reduce(v, [](float a, float b) { return fmaxf(a, b); }); }
__device__ __forceinline__ float wave_sum(float v) { return wave_reduce(v, [](float a, float b) { return a + b; }); }
// the sum over lanes l, l + STEP, l + 2 STEP, ...
template <int STEP> __device__ __forceinline__ float lanes_sum(float v)
{
    auto add = [](float a, float b) { return a + b; };
    if constexpr (STEP <= 4) v = v + dpp<0x124>(v);
    if constexpr (STEP <= 8) v = v + dpp<0x128>(v);
    if constexpr (STEP <= 16) v = across16(v, add);
    if constexpr (STEP <= 32) v = across32(v, add);
    return v;
}

// c += a b^T over 64 bytes of 16 rows each; a lane holds 16 bytes of row lane % 16.  (Which of the contracted elements a lane group holds is
// the same for both operands, so any order of them will do: rows of fp32 are read 16 bytes per lane as well and take four 16x16x4 steps.)
template <typename T> __device__ __forceinline__ void mma_rows(f32x4 &c, const u32x4 &a, const u32x4 &b);
template <> __device__ __forceinline__ void mma_rows<bf16_t>(f32x4 &c, const u32x4 &a, const u32x4 &b)
{
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ void mma_rows<f16_t>(f32x4 &c, const u32x4 &a, const u32x4 &b)
{
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ void mma_rows<float>(f32x4 &c, const u32x4 &a, const u32x4 &b)
{
#pragma unroll
    for (int t = 0; t < 4; ++t) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[t]), __uint_as_float(b[t]), c, 0, 0, 0);
}

// 16 bytes as fp32
template <typename T> struct wide { float v[vec_of<T>::n]; };
template <typename T> __device__ __forceinline__ wide<T> widen(const u32x4 &x)
{
    wide<T> r;
    if constexpr (vec_of<T>::n == 8) {
#pragma unroll
        for (int u = 0; u < 4; ++u) unpack2<T>(x[u], r.v[2 * u], r.v[2 * u + 1]);
    } else {
#pragma unroll
        for (int u = 0; u < 4; ++u) r.v[u] = __uint_as_float(x[u]);
    }
    return r;
}

// ---- sizes that kernels and host agree on ----
__host__ __device__ __forceinline__ int halo_left(int S) { return (((S - 1) / 2) + 15) & ~15; }
__host__ __device__ __forceinline__ int halo_right(int S) { return (S - 1 - (S - 1) / 2 + 15) & ~15; }
// ahead of the first column, so that the taps of a key that is a multiple of 4 begin on 16 bytes
__host__ __device__ __forceinline__ int raw_shift(int S) { return ((S - 1) / 2 - halo_left(S)) & 3; }
// columns of a row of raw scores: shift, halos, a step's keys, and what a window of whole vectors reads behind them; 12 more than a multiple
// of 16, which spreads the four row groups of an accumulator over the banks
__host__ __device__ __forceinline__ int raw_stride(int S, int nt) { return halo_left(S) + halo_right(S) + 64 * nt + 12; }
__host__ __device__ __forceinline__ int q_stride(int row_bytes) { return row_bytes + 32; }   // (conflict-free fragment reads)
__host__ __device__ __forceinline__ int up16(int x) { return (x + 15) & ~15; }

// LDS of a workgroup of the kernels that form raw scores, in bytes, part by part
struct raw_layout { int weights, raw, probs, total; };
__host__ __device__ __forceinline__ raw_layout raw_layout_of(int rows, int R, int S, int gw, int D, int size, int nt, bool attn)
{
    raw_layout l;
    const int padded = up16(rows);
    l.weights = padded * q_stride(D * size) + up16(padded * 4);
    l.raw = l.weights + up16(gw * R * ((S + 3) & ~3) * 4);
    l.probs = l.raw + up16(3 * rows * raw_stride(S, nt) * 4);
    l.total = l.probs + (attn ? DECODE_WAVES * gw * 16 * nt * 4 : 0);
    // (the wavefronts' results take the place of the raw scores at the end)
    const int results = l.raw + DECODE_WAVES * gw * (D + 2) * 4;
    if (attn && l.total < results) l.total = results;
    return l;
}

// The rows' raw scores, step by step.
template <typename T, int D, int NT> struct raw_scores {
    static constexpr int ROW = D * (int)sizeof(T), NC = ROW / 64, CH = 64 * NT;
    const decode_args &a;
    const int *entries;         // the slot's row of the table
    unsigned char *qs;          // query rows in LDS
    int *pos;                   // their positions
    float *raw;
    int rows, n, limit, kvh, lane, wave, hl, hr, stride;
    u32x4 kreg[NT][NC];
    int bad;                    // bit t: tile t lies in a page that is none

    __device__ __forceinline__ raw_scores(const decode_args &a_, unsigned char *smem, const raw_layout &l, int rows_, int b, int kvh_, int n_, int limit_)
        : a(a_), entries(a_.table + (int64_t)b * a_.max_pages), qs(smem), pos(reinterpret_cast<int *>(smem + up16(rows_) * q_stride(ROW))),
          raw(reinterpret_cast<float *>(smem + l.raw)), rows(rows_), n(n_), limit(limit_), kvh(kvh_), lane((int)threadIdx.x & 63),
          wave(__builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6)), hl(halo_left(a_.S)), hr(halo_right(a_.S)), stride(raw_stride(a_.S, NT)), bad(0)
    {
    }

    // where the rows of one 16-key tile begin in a pool; nullptr: in no page
    __device__ __forceinline__ const char *tile(const char *pool, int key0) const
    {
        const int entry = entries[key0 >> a.page_shift];
        if ((unsigned)entry >= (uint64_t)a.n_pages) return nullptr;
        const int64_t block = (int64_t)entry * a.kv_heads + kvh;
        return pool + (((block << a.page_shift) + (key0 & ((1 << a.page_shift) - 1))) * ROW);
    }
    // A tile of keys; nothing is read of one that holds none of the keys this split needs.
    __device__ __forceinline__ bool load(u32x4 (&dst)[NC], int key0) const
    {
        if (key0 < 0 || key0 >= limit) {
#pragma unroll
            for (int c = 0; c < NC; ++c) dst[c] = u32x4{0, 0, 0, 0};
            return true;
        }
        const char *at = tile(a.k, key0);
        if (!at) {
#pragma unroll
            for (int c = 0; c < NC; ++c) dst[c] = u32x4{0, 0, 0, 0};
            return false;
        }
        at += (lane & 15) * ROW + (lane >> 4) * 16;
#pragma unroll
        for (int c = 0; c < NC; ++c) dst[c] = *reinterpret_cast<const u32x4 *>(at + 64 * c);
        return true;
    }
    __device__ __forceinline__ int first_of(int kb, int t) const { return kb + hr + (wave * NT + t) * 16; }   // (a step's new keys)
    __device__ __forceinline__ void load_step(int kb)
    {
        bad = 0;
#pragma unroll
        for (int t = 0; t < NT; ++t) bad |= load(kreg[t], first_of(kb, t)) ? 0 : 1 << t;
    }
    // The scores of N tiles from key0 on, 16 query rows after 16: to column `col` of a buffer and, where they are the first columns of the next
    // step, of that one's.
    template <int N> __device__ __forceinline__ void score(const u32x4 (&kr)[N][NC], int key0, int is_bad, float *buf, int col, float *next) const
    {
        const int group = lane >> 4, at = lane & 15;
        // (all rows see all of these keys: nothing to replace)
        const bool plain = is_bad == 0 && a.window == 0 && key0 >= 0 && key0 + 16 * N - 1 <= n - a.W;
        for (int m0 = 0; m0 < rows; m0 += 16) {
            f32x4 acc[N];
#pragma unroll
            for (int t = 0; t < N; ++t) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            const unsigned char *qrow = qs + (m0 + at) * q_stride(ROW) + group * 16;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const u32x4 qv = *reinterpret_cast<const u32x4 *>(qrow + 64 * c);
#pragma unroll
                for (int t = 0; t < N; ++t) mma_rows<T>(acc[t], qv, kr[t][c]);
            }
            const int r0 = m0 + 4 * group;
            if (!plain) {
                const int4 p = *reinterpret_cast<const int4 *>(pos + r0);
                const int ps[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
                for (int t = 0; t < N; ++t)
#pragma unroll
                    for (int v = 0; v < 4; ++v) {
                        // (what a row does not see is replaced, not multiplied: garbage behind the last key stays out)
                        const int key = key0 + 16 * t + at;
                        const bool seen = key >= 0 && key <= ps[v] && (a.window == 0 || key > ps[v] - a.window);
                        acc[t][v] = !seen ? 0.0f : is_bad >> t & 1 ? __builtin_nanf("") : acc[t][v];
                    }
            }
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                if (r0 + v >= rows) break;
                float *const to = buf + (r0 + v) * stride + col + at;
#pragma unroll
                for (int t = 0; t < N; ++t) to[16 * t] = acc[t][v];
                if (next) {
#pragma unroll
                    for (int t = 0; t < N; ++t)
                        if (col + 16 * t >= CH) next[(r0 + v) * stride + col + 16 * t - CH + at] = acc[t][v];
                }
            }
        }
    }
    __device__ __forceinline__ float *buffer(int step) const { return raw + raw_shift(a.S) + (step % 3) * rows * stride; }
    // Query rows, their positions and the conv weights into LDS: rows g * W + i, position p - W + 1 + i of query head h0 + g.
    __device__ __forceinline__ void stage(unsigned char *smem, const raw_layout &l, int b, int h0) const
    {
        const int padded = up16(rows), W = a.W;
        for (int x = threadIdx.x; x < padded * (ROW / 16); x += 64 * DECODE_WAVES) {
            const int r = x / (ROW / 16), c = x % (ROW / 16), g = r / W, p = n - W + (r - g * W);
            u32x4 val = {0, 0, 0, 0};
            if (r < rows && p >= 0)
                val = *reinterpret_cast<const u32x4 *>(a.q + (((int64_t)b * a.heads + h0 + g) * a.ring + p % a.ring) * ROW + 16 * c);
            *reinterpret_cast<u32x4 *>(qs + r * q_stride(ROW) + 16 * c) = val;
            if (c == 0) pos[r] = r < rows ? p : -1;
        }
        float *w = reinterpret_cast<float *>(smem + l.weights);
        const int sp = (a.S + 3) & ~3, taps = a.R * a.S;
        for (int x = threadIdx.x; x < a.gw * taps; x += 64 * DECODE_WAVES) {
            const int g = x / taps, r = (x - g * taps) / a.S, s = x - g * taps - r * a.S;
            w[(g * a.R + r) * sp + s] = load_any(a.w, a.w_dtype, (int64_t)(h0 + g) * taps + r * a.S + s);
        }
    }
    // the tiles ahead of the first step's new keys: one per wavefront at most (four at S = 63)
    __device__ __forceinline__ void halo(int kb) const
    {
        if (wave * 16 >= hl + hr) return;
        u32x4 kr[1][NC];
        const int key0 = kb - hl + wave * 16;
        const bool ok = load(kr[0], key0);
        score<1>(kr, key0, !ok, buffer(0), wave * 16, nullptr);
    }
    // this step's scores, from the keys that load_step() brought
    __device__ __forceinline__ void score_step(int kb, int step) const
    {
        const int col = hl + hr + wave * NT * 16;
        score<NT>(kreg, first_of(kb, 0), bad, buffer(step), col, col + NT * 16 > CH ? buffer(step + 1) : nullptr);
    }
    // where the taps of the step's key `local` begin in row `row` of a buffer
    __device__ __forceinline__ const float *window(int step, int row, int local) const
    {
        return buffer(step) + row * stride + local + hl - (a.S - 1) / 2;
    }
};

// ---- the conv: a lane forms four neighbouring keys, whose taps it reads as whole vectors ----
// c[u] += sum over t < S of w[t] x[t + u]; x and w begin on 16 bytes.  Taps behind the last one are left out, not multiplied by 0 (a score may
// be infinite).  N: their number, 0: only known at run time.
template <int N> __device__ __forceinline__ void taps4(float (&c)[4], const float *x, const float *w, int S)
{
    if constexpr (N > 0) {
        constexpr int V = (N + 6) / 4;
        float xs[4 * V];
#pragma unroll
        for (int i = 0; i < V; ++i) *reinterpret_cast<f32x4 *>(xs + 4 * i) = *reinterpret_cast<const f32x4 *>(x + 4 * i);
        float ws[4 * ((N + 3) / 4)];
#pragma unroll
        for (int i = 0; i < (N + 3) / 4; ++i) *reinterpret_cast<f32x4 *>(ws + 4 * i) = *reinterpret_cast<const f32x4 *>(w + 4 * i);
#pragma unroll
        for (int t = 0; t < N; ++t)
#pragma unroll
            for (int u = 0; u < 4; ++u) c[u] = fmaf(ws[t], xs[t + u], c[u]);
    } else {
        f32x4 lo = *reinterpret_cast<const f32x4 *>(x);
        for (int t0 = 0; t0 < S; t0 += 4) {
            const f32x4 hi = *reinterpret_cast<const f32x4 *>(x + t0 + 4), wv = *reinterpret_cast<const f32x4 *>(w + t0);
            const float xs[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
            for (int t = 0; t < 4; ++t)
                if (t0 + t < S) {
#pragma unroll
                    for (int u = 0; u < 4; ++u) c[u] = fmaf(wv[t], xs[t + u], c[u]);
                }
            lo = hi;
        }
    }
}
template <int N> struct count_of { static constexpr int value = N; };
// f(count_of<S>) for the sizes with unrolled code, f(count_of<0>) for the others
template <typename F> __device__ __forceinline__ void with_taps(int S, F f)
{
    switch (S) {
    case 3: f(count_of<3>()); break;
    case 5: f(count_of<5>()); break;
    case 7: f(count_of<7>()); break;
    case 9: f(count_of<9>()); break;
    case 11: f(count_of<11>()); break;
    case 15: f(count_of<15>()); break;
    default: f(count_of<0>()); break;
    }
}
// Four values per lane, for the keys 4 * (lane % (4 NT)) .. + 3, partial over the lanes of equal lane % (4 NT): the whole sum of key
// 4 * (lane % (4 NT)) + lane / 16 in every lane.  Halves and rows change places as they are added, so a value is moved once and not four times.
template <int NT> __device__ __forceinline__ float deal4(float (&c)[4])
{
    swap32(c[0], c[2]);
    swap32(c[1], c[3]);
    uint32_t p = __float_as_uint(c[0] + c[2]), q = __float_as_uint(c[1] + c[3]);   // lower half: keys 0 and 1, upper half: 2 and 3
    swap16(p, q);
    float v = __uint_as_float(p) + __uint_as_float(q);
    if constexpr (NT <= 2) v += dpp<0x128>(v);
    if constexpr (NT == 1) v += dpp<0x124>(v);
    return v;
}

// A wavefront's 16 * NT rows of V times the probabilities of GW heads: a row is read by ROW / 16 lanes.
template <typename T, int D, int NT, int GW> struct value_rows {
    static constexpr int ROW = D * (int)sizeof(T), LPR = ROW / 16, RPI = 64 / LPR, NV = 16 * NT / RPI, E = vec_of<T>::n;
    u32x4 vreg[NV];
    float acc[GW][E];

    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int g = 0; g < GW; ++g)
#pragma unroll
            for (int e = 0; e < E; ++e) acc[g][e] = 0.0f;
    }
    // rows first .. first + 16 NT - 1; zeros for those outside lo .. end - 1.  tile(key) gives a tile's place, or nullptr
    template <typename F> __device__ __forceinline__ void load(int first, int lo, int end, int lane, F tile)
    {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int key0 = first + 16 * t;
            const char *at = key0 < end && key0 + 15 >= lo ? tile(key0) : nullptr;
#pragma unroll
            for (int i = 0; i < 16 / RPI; ++i) {
                const int row = i * RPI + lane / LPR;
                u32x4 x = {0, 0, 0, 0};
                if (at && key0 + row >= lo && key0 + row < end) x = *reinterpret_cast<const u32x4 *>(at + row * ROW + (lane % LPR) * 16);
                vreg[t * (16 / RPI) + i] = x;
            }
        }
    }
    // probs: the wavefront's rows, 16 NT of each head
    __device__ __forceinline__ void multiply(const float *probs, int lane)
    {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const wide<T> x = widen<T>(vreg[i]);
#pragma unroll
            for (int g = 0; g < GW; ++g) {
                const float p = probs[g * 16 * NT + i * RPI + lane / LPR];
#pragma unroll
                for (int e = 0; e < E; ++e) acc[g][e] = fmaf(p, x.v[e], acc[g][e]);
            }
        }
    }
    // the sums over the row groups, to dst[g][D]
    __device__ __forceinline__ void store(float *dst, int lane)
    {
#pragma unroll
        for (int g = 0; g < GW; ++g)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float s = lanes_sum<LPR>(acc[g][e]);
                if (lane < LPR) dst[g * D + lane * E + e] = s;
            }
    }
};

// ---- host side ----
inline int check_cache(const mta_cache *c)
{
    if (!c || !c->k || !c->v || !c->q || !c->table || !c->state) return MTA_ERR_NULL;
    if (dtype_size(c->dtype) == 0) return MTA_ERR_DTYPE;
    if (c->n_pages <= 0 || c->n_pages > INT32_MAX || c->slots <= 0 || c->slots > 65535 || c->max_pages <= 0 || c->heads <= 0 || c->heads > 4096 || c->kv_heads <= 0
        || c->query_rows <= 0 || c->query_rows > 65535)
        return MTA_ERR_SHAPE;
    if (c->page < 16 || c->page > 1024 || (c->page & (c->page - 1)) || (int64_t)c->max_pages * c->page > (1 << 30)) return MTA_ERR_SHAPE;
    if (c->heads % c->kv_heads) return MTA_ERR_GROUP;
    if (c->head_dim != 64 && c->head_dim != 128) return MTA_ERR_HEAD_DIM;
    if (!aligned_to(c->k, 16) || !aligned_to(c->v, 16) || !aligned_to(c->q, 16) || !aligned_to(c->table, 4) || !aligned_to(c->state, 4)) return MTA_ERR_ALIGN;
    return MTA_OK;
}
inline int page_shift_of(int page)
{
    int s = 0;
    while ((1 << s) < page) ++s;
    return s;
}
inline decode_args args_of(const mta_cache *c, const void *w, int R, int S, int out_rows, int window, int64_t longest, float scale, int w_dtype)
{
    decode_args a = {};
    a.k = (const char *)c->k, a.v = (const char *)c->v, a.q = (const char *)c->q, a.w = w, a.table = c->table, a.state = c->state;
    a.n_pages = c->n_pages, a.slots = c->slots, a.max_pages = c->max_pages, a.page_shift = page_shift_of(c->page);
    a.heads = c->heads, a.kv_heads = c->kv_heads, a.share = c->heads / c->kv_heads, a.ring = c->query_rows;
    a.R = R, a.S = S, a.W = R + out_rows - 1, a.window = window, a.longest = (int)longest, a.scale = scale, a.w_dtype = w_dtype;
    return a;
}
// keys that the splits of one slot have to cover at most
inline int64_t span_of(int64_t longest, int window, int out_rows)
{
    const int64_t seen = window > 0 ? (int64_t)window + out_rows - 1 + 15 : longest;
    return seen < longest ? seen : longest;
}
template <typename K> inline int allow_lds(K kern, int bytes)
{
    if (bytes <= 64 << 10) return MTA_OK;
    const hipError_t e = hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    return e == hipSuccess ? MTA_OK : (int)e;
}

}  // namespace mta
