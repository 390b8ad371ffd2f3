// What the kernels of single-token attention over a paged cache share (decode_attn.hip, decode_mta.hip).
//
// A slot b holds n tokens: the ones it had (state[0][b]) and the ones it got last (state[1][b]; none: the slot sits this step out).  The newest
// query row is p = n - 1.  Keys and values lie in pages (page, key head, row, element), table[b][key / page] names the page; queries in a
// ring, position i in row i % ring.  A row i sees the keys max(0, i - window + 1) .. i; what a row does not see counts as 0 ahead of the conv.
//
// Work split.  A workgroup of four wavefronts takes one slot, one or more query heads of one key head, and a stretch of the keys (an "item",
// see shares), in steps of 64 * NT keys, 16 * NT per wavefront.  Keys are tiles of 16 consecutive rows of a page, read straight into the operand
// fragments of 16x16 products (no key is used by two wavefronts, so LDS would only add a pass); the query rows that the conv needs, one to a
// few tens, are the other operand, in LDS.  The conv takes what it needs of neighbouring keys from LDS, where the last columns of a step are
// written a second time, as the first columns of the next one: keys are read twice only where an item begins (halo).  Three buffers of raw
// scores: one is read, the next one gets the columns to come, and the one before may still be read by a wavefront that is behind - a single
// barrier per step.
//
// What bounds it: K and V are read once, 2 D elements per key and head against some 2 R D + 2 R S + 2 D operations on them, so memory - where the
// keys are many.  Below some megabytes it is the chain from the state to the table to K to LDS to the result, 4 to 6 us a kernel.
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
    int target, least, items;   // how the slots' keys are shared out (shares)
    int gw;                     // query heads per workgroup
    float scale;
};

// One slot's step: n < 0: not a state of this cache, or more tokens than grid and workspace were sized for (its outputs are NaN); 0: it
// sits this step out (zeros).  older: output rows ahead of the newest one.
// base: where the items begin, a multiple of 16; lo: the first key that the newest row sees.
struct slot_step { int n, base, lo; };
__device__ __forceinline__ slot_step step_of(const decode_args &a, int b, int older)
{
    const int had = a.state[b], got = a.state[a.slots + b];
    slot_step s = {0, 0, 0};
    if (had < 0 || got < 0 || (got > 0 && had > a.longest - got)) { s.n = -1; return s; }   // (had + got may pass 32 bits)
    if (got == 0) return s;
    s.n = had + got;
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
    if constexpr (STEP <= 8) v = v + dpp<0x128>(v);
    if constexpr (STEP <= 16) v = across16(v, add);
    if constexpr (STEP <= 32) v = across32(v, add);
    return v;
}

template <int CTRL, int ROWS> __device__ __forceinline__ int dpp_or_0(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, true); }
// the sum over the lanes up to this one: within rows of 16, then the rows' last sums onto the rows behind them
__device__ __forceinline__ int wave_scan(int v)
{
    v += dpp_or_0<0x111, 0xf>(v);
    v += dpp_or_0<0x112, 0xf>(v);
    v += dpp_or_0<0x114, 0xf>(v);
    v += dpp_or_0<0x118, 0xf>(v);
    v += dpp_or_0<0x142, 0xa>(v);
    v += dpp_or_0<0x143, 0xc>(v);
    return v;
}

// How the slots' keys are shared out over workgroups.  The host knows the longest slot at most (a captured graph: not even that), so the
// device does it: every slot's keys in steps, `per` of them to an item.  Items of one size, however different the lengths, and all that live
// next to each other in the grid, which deals its workgroups over the XCDs in turn: with a grid of (split, head, slot) short slots left
// whole XCDs idle (conv-attention, 16 slots of 1k to 8k keys 204 us that way, 153 this way; MTA, 16 slots of 512 to 4k keys 142, 84).
// per: `target` items are one round of workgroups that are all resident (an item costs some 5 us beside its keys - the table, queries, weights,
// the first loads, the results - which a second round pays again: 8k keys of 32 heads 30 us in one round, 37 in two); where they come
// out long, four times as many, which even out the end (16 slots of up to 8k keys 165 us in items of 25 steps, 153 in 7).
// A slot has an item at least: somebody writes its result.  Every wavefront computes this for itself, a slot to a lane.
struct shares {
    const decode_args &a;
    const int older, shift;     // output rows ahead of the newest one; log2 of the keys of a step
    const bool newest;          // the keys of the newest row only, not of all output rows
    int per;
    slot_step mine;             // of the first 64 slots, one to a lane
    static constexpr int LONG = 8, SHORT = 6, MORE = 4;

    __device__ __forceinline__ int from(const slot_step &s) const { return newest ? s.lo & ~15 : s.base; }
    __device__ __forceinline__ int steps(const slot_step &s) const { return s.n > 0 ? (s.n - from(s) + (1 << shift) - 1) >> shift : 0; }
    __device__ __forceinline__ slot_step slot(int b) const
    {
        slot_step s = {0, 0, 0};
        if (b < a.slots) s = step_of(a, b, older);
        return s;
    }
    __device__ __forceinline__ shares(const decode_args &a_, int older_, int shift_, bool newest_, int lane)
        : a(a_), older(older_), shift(shift_), newest(newest_), mine(slot(lane))
    {
        float total = (float)steps(mine);     // (of up to 2^40 steps; the same in every wavefront)
        for (int b0 = 64; b0 < a.slots; b0 += 64) total += (float)steps(slot(b0 + lane));
        total = wave_sum(total);
        per = (int)ceilf(total / (float)a.target);
        if (per > LONG) {
            per = (int)ceilf(total / (float)(MORE * a.target));
            if (per < SHORT) per = SHORT;
        }
        if (per < a.least) per = a.least;
    }
    __device__ __forceinline__ int items(int b, const slot_step &s) const
    {
        const int n = (int)((unsigned)(steps(s) + per - 1) / (unsigned)per);
        return b >= a.slots ? 0 : n > 1 ? n : 1;
    }
};
// Item `index` (or, slot >= 0, the first one of that slot): its slot's step, the slot's first item and their number; slot < 0: there is no such item.
struct work_item { slot_step s; int slot, first, count; };
__device__ __forceinline__ work_item item_of(const shares &sh, int index, int slot, int lane)
{
    work_item w;
    int before = 0;
    slot_step s = sh.mine;
    for (int b0 = 0; b0 < sh.a.slots; b0 += 64) {
        if (b0 > 0) s = sh.slot(b0 + lane);
        const int n = sh.items(b0 + lane, s), upto = before + wave_scan(n);
        const uint64_t behind = __ballot(slot >= 0 ? b0 + lane >= slot : upto > index);
        if (behind) {
            const int l = __builtin_ctzll(behind);
            w.slot = b0 + l;
            w.count = __builtin_amdgcn_readlane(n, l);
            w.first = __builtin_amdgcn_readlane(upto, l) - w.count;
            w.s.n = __builtin_amdgcn_readlane(s.n, l), w.s.base = __builtin_amdgcn_readlane(s.base, l), w.s.lo = __builtin_amdgcn_readlane(s.lo, l);
            return w;
        }
        before = __builtin_amdgcn_readlane(upto, 63);
    }
    w.slot = -1;
    return w;
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

// 64 entries of a slot's row of the table, one per lane, from the page of `key` on: one load and one wait for all the tiles they serve.  (An entry
// at a time was a chain of waits ahead of the first loads of K and V: 14k of a workgroup's 31k cycles at 8k keys of 32 heads.)
struct page_map {
    int first, entry;
    __device__ __forceinline__ void load(const decode_args &a, int b, int key, int lane)
    {
        first = (key > 0 ? key : 0) >> a.page_shift;
        const int i = first + lane;
        entry = a.table[(int64_t)b * a.max_pages + (i < a.max_pages ? i : a.max_pages - 1)];
    }
    // ... from the page of `key` on, if those up to that of `last` are not there
    __device__ __forceinline__ void reach(const decode_args &a, int b, int key, int last, int lane)
    {
        if ((last >> a.page_shift) - first >= 64) load(a, b, key, lane);
    }
    // Where a lane's bytes (at `offset` from the tile's first row of ROW bytes) of the tile at key0 lie in a pool.  Of a tile that is not wanted, or
    // whose entry names no page (ok = false), all lanes get the pool's first bytes, which the caller does not use: loads without branches
    // around them stay in flight behind each other (with branches the wait for one was a wait for all), and one line costs next to nothing.
    template <int ROW> __device__ __forceinline__ const char *tile(const decode_args &a, int kvh, const char *pool, int key0, int offset, bool wanted, bool &ok) const
    {
        const int e = __builtin_amdgcn_readlane(entry, wanted ? (key0 >> a.page_shift) - first : 0);
        ok = (unsigned)e < (uint64_t)a.n_pages;
        const bool there = ok && wanted;
        const int64_t block = there ? (int64_t)e * a.kv_heads + kvh : 0;
        return pool + ((block << a.page_shift) + (there ? key0 & ((1 << a.page_shift) - 1) : 0)) * ROW + (there ? offset : 0);
    }
};

// The rows' raw scores, step by step.
template <typename T, int D, int NT> struct raw_scores {
    static constexpr int ROW = D * (int)sizeof(T), NC = ROW / 64, CH = 64 * NT;
    const decode_args &a;
    page_map pages;
    unsigned char *qs;          // query rows in LDS
    int *pos;                   // their positions
    float *raw;
    int rows, n, limit, kvh, lane, wave, hl, hr, stride;
    u32x4 kreg[NT][NC];
    int bad;                    // bit t: tile t lies in a page that is none

    __device__ __forceinline__ raw_scores(const decode_args &a_, unsigned char *smem, const raw_layout &l, const page_map &pages_, int rows_, int kvh_, int n_, int limit_)
        : a(a_), pages(pages_), qs(smem), pos(reinterpret_cast<int *>(smem + up16(rows_) * q_stride(ROW))),
          raw(reinterpret_cast<float *>(smem + l.raw)), rows(rows_), n(n_), limit(limit_), kvh(kvh_), lane((int)threadIdx.x & 63),
          wave(__builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6)), hl(halo_left(a_.S)), hr(halo_right(a_.S)), stride(raw_stride(a_.S, NT)), bad(0)
    {
    }

    // A tile of keys, if it holds any that this item needs; false: it lies in no page.
    __device__ __forceinline__ bool load(u32x4 (&dst)[NC], int key0, bool wanted = true) const
    {
        bool ok;
        wanted = wanted && key0 >= 0 && key0 < limit;
        const char *at = pages.tile<ROW>(a, kvh, a.k, key0, (lane & 15) * ROW + (lane >> 4) * 16, wanted, ok);
#pragma unroll
        for (int c = 0; c < NC; ++c) dst[c] = *reinterpret_cast<const u32x4 *>(at + 64 * c);
        return ok || !wanted;
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
        int m0 = 0;
        do {   // (at least once, which the compiler has to know to keep other loads in flight)
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
        } while ((m0 += 16) < rows);
    }
    __device__ __forceinline__ float *buffer(int step) const { return raw + raw_shift(a.S) + (step % 3) * rows * stride; }
    // What precedes the first step.  begin(): the loads of the tiles ahead of its new keys (one per wavefront at most, four at S = 63), of the query
    // rows and of the weights, ahead of the first step's own; finish(): query rows (g * W + i: position p - W + 1 + i of query head h0 + g), their
    // positions and weights to LDS, and the scores of those tiles.
    struct start {
        u32x4 halo[1][NC], q[2];
        float w[2];
        bool halo_ok;
    };
    __device__ __forceinline__ int position(int r) const { return r < rows ? n - a.W + r % a.W : -1; }
    __device__ __forceinline__ u32x4 query(int x, int b, int h0) const
    {
        const int r = x / (ROW / 16), c = x % (ROW / 16), g = r / a.W, p = position(r);
        u32x4 val = {0, 0, 0, 0};
        if (p >= 0) val = *reinterpret_cast<const u32x4 *>(a.q + (((int64_t)b * a.heads + h0 + g) * a.ring + p % a.ring) * ROW + 16 * c);
        return val;
    }
    __device__ __forceinline__ void begin(start &st, int kb, int b, int h0) const
    {
        const int taps = a.gw * a.R * a.S, tid = threadIdx.x;
        const int64_t w0 = (int64_t)h0 * a.R * a.S;
        st.halo_ok = load(st.halo[0], kb - hl + wave * 16, wave * 16 < hl + hr);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            st.q[u] = query(tid + 256 * u, b, h0);
            st.w[u] = load_any(a.w, a.w_dtype, w0 + (tid + 256 * u < taps ? tid + 256 * u : 0));
        }
    }
    __device__ __forceinline__ void finish(const start &st, int kb, int b, int h0, unsigned char *smem, const raw_layout &l) const
    {
        const int vecs = up16(rows) * (ROW / 16), taps = a.gw * a.R * a.S, sp = (a.S + 3) & ~3, tid = threadIdx.x;
        const int64_t w0 = (int64_t)h0 * a.R * a.S;
        float *const w = reinterpret_cast<float *>(smem + l.weights);
        auto put = [&](int x, const u32x4 &val, int p) {
            *reinterpret_cast<u32x4 *>(qs + x / (ROW / 16) * q_stride(ROW) + x % (ROW / 16) * 16) = val;
            if (x % (ROW / 16) == 0) pos[x / (ROW / 16)] = p;
        };
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int x = tid + 256 * u;
            if (x < vecs) put(x, st.q[u], position(x / (ROW / 16)));
            if (x < taps) w[x / a.S * sp + x % a.S] = st.w[u];
        }
        for (int x = tid + 512; x < vecs; x += 256) put(x, query(x, b, h0), position(x / (ROW / 16)));
        for (int x = tid + 512; x < taps; x += 256) w[x / a.S * sp + x % a.S] = load_any(a.w, a.w_dtype, w0 + x);
        __syncthreads();
        if (wave * 16 < hl + hr) score<1>(st.halo, kb - hl + wave * 16, !st.halo_ok, buffer(0), wave * 16, nullptr);
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
constexpr int log2_of(int x) { return x > 1 ? 1 + log2_of(x >> 1) : 0; }
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
// How a wavefront's 64 lanes share 16 NT keys of GW heads, four keys to a lane: quad (4 NT of them), head, and the rows of taps, dealt over RG
// lanes.  deal() adds the RG parts and leaves each lane VALUES whole sums, of keys first .. first + VALUES - 1 of its quad: halves and rows of
// lanes change places as they are added, so a value is moved once.  With RG > 4 several lanes hold the same key, one of them is its owner.
template <int NT, int GW> struct score_lanes {
    static constexpr int QUADS = 4 * NT, RG = 16 / (NT * GW), VALUES = RG == 1 ? 4 : RG == 2 ? 2 : 1;
    int quad, head, part, key;
    bool owner;
    __device__ __forceinline__ explicit score_lanes(int lane)
        : quad(lane % QUADS), head(lane / QUADS % GW), part(lane / (QUADS * GW)),
          key(4 * (lane % QUADS) + (RG == 1 ? 0 : RG == 2 ? 2 * (lane >> 5) : lane >> 4)), owner(RG <= 4 || lane / (QUADS * GW) % (RG / 4 + (RG < 4)) == 0)
    {
    }
    __device__ __forceinline__ void deal(float (&c)[4]) const
    {
        if constexpr (RG >= 2) {
            swap32(c[0], c[2]);
            swap32(c[1], c[3]);
            c[0] += c[2], c[1] += c[3];   // lower half: keys 0 and 1, upper half: 2 and 3
        }
        if constexpr (RG >= 4) {
            uint32_t p = __float_as_uint(c[0]), q = __float_as_uint(c[1]);
            swap16(p, q);
            c[0] = __uint_as_float(p) + __uint_as_float(q);
        }
        if constexpr (RG >= 8) c[0] += dpp<0x128>(c[0]);
        if constexpr (RG == 16) c[0] += dpp<0x124>(c[0]);
    }
    // over all lanes of the same head
    template <typename F> __device__ __forceinline__ static float reduce(float v, F op)
    {
        v = op(v, dpp<0xb1>(v));
        v = op(v, dpp<0x4e>(v));
        if constexpr (!(QUADS == 4 && GW >= 2)) v = op(v, dpp<0x141>(v));
        if constexpr (!((QUADS == 4 && GW == 4) || (QUADS == 8 && GW >= 2))) v = op(v, dpp<0x128>(v));
        if constexpr (!((QUADS == 8 && GW == 4) || (QUADS == 16 && GW >= 2))) v = across16(v, op);
        if constexpr (!(QUADS == 16 && GW == 4)) v = across32(v, op);
        return v;
    }
};

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
    // rows first .. first + 16 NT - 1, as far as they lie in lo .. end - 1
    __device__ __forceinline__ void load(const decode_args &a, const page_map &pages, int kvh, int first, int lo, int end, int lane)
    {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            bool ok;
            const int key0 = first + 16 * t;
            const char *at = pages.tile<ROW>(a, kvh, a.v, key0, lane / LPR * ROW + lane % LPR * 16, key0 < end && key0 + 15 >= lo, ok);
#pragma unroll
            for (int i = 0; i < 16 / RPI; ++i) vreg[t * (16 / RPI) + i] = *reinterpret_cast<const u32x4 *>(at + i * RPI * ROW);
            // (a page that is none: its keys' probabilities are NaN)
        }
    }
    // the same rows times probs, 16 NT of each head
    __device__ __forceinline__ void multiply(const float *probs, int first, int lo, int end, int lane)
    {
        if (first < lo || first + 16 * NT > end) {   // (replaced, not multiplied by 0: what lies there may be anything)
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int key = first + i * RPI + lane / LPR;
                if (key < lo || key >= end) vreg[i] = u32x4{0, 0, 0, 0};
            }
        }
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
// keys that the items of one slot have to cover at most
inline int64_t span_of(int64_t longest, int window, int out_rows)
{
    const int64_t seen = window > 0 ? (int64_t)window + out_rows - 1 + 15 : longest;
    return seen < longest ? seen : longest;
}
// Keys per step and wavefront, in tiles of 16: 8 KB of K and as many of V.  More in flight is slower, not faster: a kernel that only reads pages
// this way gets 5.8 to 6.1 TB/s with one or two tiles of 256-byte rows and 4.6 with four, whatever the number of workgroups.
constexpr int most_tiles(int row_bytes) { return row_bytes >= 512 ? 1 : 512 / row_bytes; }
// Keys per step (64 nt, nt up to `most`), and what `shares` goes by; `groups` workgroups take an item, one of them for some heads each.  `round`
// workgroups are one round: two to a CU with the registers for K and V, four without; of the shortest steps four.  A round of which each had
// fewer than four steps takes shorter ones.  Slots of a few steps stay whole where there are many of them and their results would have to be
// joined (conv-attention, us, shared out | whole: 16 slots x 16 heads of 256 keys 17.0 | 10.6, of 512 22.2 | 14.8, of 1024 28.5 | 23.8; 1 slot of
// 512 10.4 | 12.7).
struct cut { int nt, target, least, items; bool joined; };
inline cut cut_of(int64_t span, int64_t slots, int64_t groups, int most, int round, bool joins)
{
    cut c = {};
    for (c.nt = most; c.nt >= 1; c.nt >>= 1) {
        const int64_t steps = (span + 64 * c.nt - 1) / (64 * c.nt), resident = c.nt == 1 ? 1024 : round;
        c.target = (int)(resident / groups > 1 ? resident / groups : 1);
        const bool whole = joins && (steps <= 2 || (steps <= 8 && 32 * steps <= slots * groups));
        if (c.nt > 1 && (whole ? span <= 32 * c.nt : steps * slots < 4 * c.target)) continue;
        c.least = whole ? (int)steps : c.nt == 1 ? 1 : 2;
        c.joined = steps > c.least;   // (else no slot has more than one item)
        const int64_t most_items = (steps * slots > (int64_t)shares::LONG * c.target ? shares::MORE * c.target : c.target) + slots + 1;
        const int64_t all = slots * ((steps + c.least - 1) / c.least);
        c.items = (int)(all < most_items ? all : most_items);
        break;
    }
    return c;
}
template <typename K> inline int allow_lds(K kern, int bytes)
{
    if (bytes <= 64 << 10) return MTA_OK;
    const hipError_t e = hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    return e == hipSuccess ? MTA_OK : (int)e;
}
// (a launch has fewer than 2^32 threads)
inline bool too_many(const cut &c, int64_t groups) { return c.items * groups >= 1 << 24; }

}  // namespace mta
