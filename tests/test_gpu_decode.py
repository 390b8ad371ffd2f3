"""Single-token attention over a paged cache on the GPU, against whole sequences in 64 bits (tests/decode_oracle.py)."""
import math

import pytest
import torch

import multitokenatention_triton_amd as mta
from multitokenatention_triton_amd import ops

from decode_oracle import check, token

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


class Sequences:
    """Whole sequences on the host, and a cache that is fed from them."""

    def __init__(self, lengths, h, hkv, d, dtype, page, rows, seed=0, n_pages=None, max_pages=None, scatter=True):
        g = torch.Generator().manual_seed(seed)
        self.h, self.hkv, self.d, self.dtype, self.gen = h, hkv, d, dtype, g
        most = max(max(lengths), 1) + 8
        self.q = torch.randn(len(lengths), h, most, d, generator=g).to(dtype)
        self.k = torch.randn(len(lengths), hkv, most, d, generator=g).to(dtype)
        self.v = torch.randn(len(lengths), hkv, most, d, generator=g).to(dtype)
        need = -(-most // page)
        self.cache = mta.PagedCache(len(lengths), n_pages or len(lengths) * need + 5, h, d, hkv, page, max_pages or need + 1, rows, dtype)
        for pool in (self.cache.k, self.cache.v, self.cache.q):
            pool.fill_(float("nan"))           # nothing that was not appended may be used
        # pages in the order in which slots happen to need them
        if scatter:
            left = list(lengths)
            while any(left):
                now = [min(n, page) if torch.rand(1, generator=g) < 0.6 else 0 for n in left]
                if any(now):
                    self.feed(now)
                left = [n - c for n, c in zip(left, now)]
        else:
            self.feed(lengths)

    def feed(self, counts):
        """The next counts[b] tokens of each sequence."""
        had = self.cache.lengths
        self.cache.extend(counts)
        n = max(counts)
        new = [torch.stack([torch.nn.functional.pad(x[b, :, had[b]:had[b] + c], (0, 0, 0, n - c), value=float("nan")) for b, c in enumerate(counts)]).cuda()
               for x in (self.q, self.k, self.v)]
        self.cache.append(*new)

    def want(self, b, w, scale, **more):
        n = self.cache.lengths[b]
        more = {name: x.double() if isinstance(x, torch.Tensor) else x for name, x in more.items()}
        return token(self.q[b, :, :n].double(), self.k[b, :, :n].double(), self.v[b, :, :n].double(), w.double(), scale, **more)


def conv_weight(h, r, s, dtype, g):
    w = 0.2 * torch.randn(h, r, s, generator=g)
    w[:, r - 1, (s - 1) // 2] += 1.0
    return w.to(dtype)


def head_weight(h, group, dtype, g):
    w = torch.eye(h) + 0.2 * torch.randn(h, h, generator=g)
    return (w * torch.block_diag(*[torch.ones(group, group)] * (h // group))).to(dtype)


def conv_module(w):
    module = mta.TritonConvAttention(w.size(0), tuple(w.shape[1:]), causal=True).to("cuda", w.dtype)
    with torch.no_grad():
        module.weight.copy_(w)
    return module


def mta_module(w, pre, w2, post, **declared):
    h = w.size(0)
    sizes = tuple(w2.shape[1:]) if w2 is not None else (3, 3)
    config = mta.MTAConfig(query_kernel_size=w.size(1), key_kernel_size=w.size(2), after_sm_query_kernel_size=sizes[0], after_sm_key_kernel_size=sizes[1])
    module = mta.MTAAttentionTriton(h, config, dropout=0.0, causal=True).to("cuda", w.dtype)
    module.reset_mta_parameters()
    with torch.no_grad():
        module.mta_conv_triton.weight.copy_(w)
        if w2 is not None:
            module.mta_conv_after_sm_triton.weight.copy_(w2)
        if pre is not None:
            module.wpsm_triton.weight.copy_(pre)
        if post is not None:
            module.wposm_triton.weight.copy_(post)
    if declared:
        module.declare_weight_structure(**declared)
    return module


LENGTHS = [[1, 2, 15, 16, 17], [33, 0, 300, 64, 5], [1001]]


# ---- fused conv-attention --------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("h,hkv,r,s,page,lengths", [
    (4, 4, 3, 5, 16, LENGTHS[0]), (4, 4, 6, 11, 64, LENGTHS[1]), (8, 2, 6, 11, 32, LENGTHS[1]), (12, 4, 5, 7, 16, LENGTHS[2]), (2, 1, 1, 1, 64, LENGTHS[1]),
    (4, 2, 11, 15, 128, LENGTHS[1]), (1, 1, 2, 4, 16, LENGTHS[2]), (4, 1, 32, 63, 16, LENGTHS[1]), (16, 16, 7, 9, 256, LENGTHS[2]), (3, 3, 4, 33, 32, LENGTHS[2])])
def test_conv_attention(dtype, d, h, hkv, r, s, page, lengths):
    print(f"conv decode {dtype} d={d} h={h}/{hkv} {r}x{s} page={page} {lengths}", flush=True)
    seq = Sequences(lengths, h, hkv, d, dtype, page, r)
    w = conv_weight(h, r, s, dtype, seq.gen)
    module = conv_module(w)
    assert module.decode_query_rows == r
    # one more token for all but the last slot
    new = [1] * len(lengths)
    new[-1] = 0 if len(lengths) > 1 else 1
    seq.feed(new)
    got = module.decode(seq.cache, 0.3)
    assert got.shape == (len(lengths), h, 1, d) and got.dtype == dtype
    for b, c in enumerate(new):
        if c == 0:
            assert torch.equal(got[b], torch.zeros_like(got[b]))
            continue
        check(got[b, :, 0], *seq.want(b, w, 0.3), what=f"slot {b}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [1, 2, 16, 100, 5000])
def test_conv_attention_window(dtype, window):
    seq = Sequences([1, 16, 99, 513, 700], 4, 2, 64, dtype, 32, 6)
    w = conv_weight(4, 6, 11, dtype, seq.gen)
    got = conv_module(w).decode(seq.cache, window=window)
    had = [c for c in seq.cache._added]
    for b, c in enumerate(had):
        if c:
            check(got[b, :, 0], *seq.want(b, w, 64 ** -0.5, window=window), what=f"slot {b}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_long_cache_in_many_splits(dtype):
    """Several steps per split, several splits, 16 wavefronts' worth of statistics; weights of another dtype."""
    seq = Sequences([9001, 4100], 8, 2, 64, dtype, 64, 6, scatter=False)
    w = conv_weight(8, 6, 11, torch.float32, seq.gen)
    got = conv_module(w).decode(seq.cache)
    for b in range(2):
        check(got[b, :, 0], *seq.want(b, w, 64 ** -0.5), what=f"slot {b}")


@pytest.mark.parametrize("h,hkv,n_slots,length", [(32, 32, 3, 2100), (32, 8, 9, 1100), (16, 16, 40, 310)])
def test_many_workgroups(h, hkv, n_slots, length):
    """Grids that are large enough for long steps."""
    seq = Sequences([length - 7 * b for b in range(n_slots)], h, hkv, 64, torch.bfloat16, 64, 5, scatter=False)
    w = conv_weight(h, 5, 7, torch.bfloat16, seq.gen)
    got = conv_module(w).decode(seq.cache)
    for b in range(0, n_slots, 4):
        check(got[b, :, 0], *seq.want(b, w, 64 ** -0.5), what=f"slot {b}")


@pytest.mark.parametrize("h,hkv,d,page,n_slots,length,dtype", [
    (32, 32, 64, 16, 40, 1500, torch.bfloat16),     # items of more than 64 pages
    (8, 8, 64, 16, 70, 900, torch.float32),         # more slots than lanes, more pages than entries at a time
    (4, 1, 128, 32, 130, 200, torch.float16),       # ... whole slots
    (16, 4, 128, 16, 9, 2500, torch.bfloat16)])
def test_slots_of_all_lengths(h, hkv, d, page, n_slots, length, dtype):
    """Keys shared out over slots of very different lengths, some empty, some that sit the step out."""
    g = torch.Generator().manual_seed(5)
    lengths = [int(length * x) for x in torch.rand(n_slots, generator=g).pow(2).tolist()]
    lengths[3], lengths[-1] = length, 0
    seq = Sequences(lengths, h, hkv, d, dtype, page, 7, scatter=False)
    w, w2 = conv_weight(h, 4, 5, dtype, seq.gen), conv_weight(h, 3, 3, dtype, seq.gen)
    pre, post = head_weight(h, 4, dtype, seq.gen), head_weight(h, 4, dtype, seq.gen)
    seq.feed([1 if b % 5 != 2 else 0 for b in range(n_slots)])
    got = conv_module(w).decode(seq.cache), mta_module(w, pre, w2, post).decode(seq.cache)
    for b in list(range(0, n_slots, 1 + n_slots // 8)) + [2, 3, n_slots - 1]:
        if b % 5 == 2:
            assert not got[0][b].any() and not got[1][b].any()
            continue
        check(got[0][b, :, 0], *seq.want(b, w, d ** -0.5), what=f"slot {b}")
        check(got[1][b, 0], *seq.want(b, w, d ** -0.5, pre=pre, w2=w2, post=post), what=f"slot {b}")


# ---- Multi-Token Attention ---------------------------------------------------------------------------------------------------
MTA = [  # h, hkv, r, s, r2, s2, group (0: dense), page, lengths
    (4, 4, 3, 3, 3, 3, 0, 16, LENGTHS[0]), (8, 8, 6, 11, 0, 0, 4, 64, LENGTHS[1]), (8, 2, 6, 11, 3, 5, 2, 32, LENGTHS[1]), (16, 16, 7, 7, 7, 7, 0, 64, LENGTHS[2]),
    (12, 6, 5, 7, 2, 9, 6, 16, LENGTHS[1]), (4, 2, 11, 15, 11, 15, 0, 64, LENGTHS[1]), (2, 1, 1, 1, 1, 3, 0, 16, LENGTHS[2]), (4, 4, 4, 33, 5, 63, 0, 16, LENGTHS[1]),
    (40, 8, 3, 3, 0, 0, 20, 32, LENGTHS[1]), (32, 32, 3, 3, 3, 3, 0, 32, LENGTHS[1]), (2, 2, 32, 63, 32, 63, 0, 16, [200, 31])]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("case", MTA)
def test_mta(dtype, d, case):
    h, hkv, r, s, r2, s2, group, page, lengths = case
    print(f"mta decode {dtype} d={d} {case}", flush=True)
    seq = Sequences(lengths, h, hkv, d, dtype, page, r + max(r2, 3) - 1)
    w, w2 = conv_weight(h, r, s, dtype, seq.gen), conv_weight(h, r2, s2, dtype, seq.gen) if r2 else None
    pre, post = head_weight(h, group or h, dtype, seq.gen), head_weight(h, group or h, dtype, seq.gen)
    declared = dict(pre_head_group=group, post_head_group=group, post_conv_identity=not r2) if group else {}
    module = mta_module(w, pre, w2, post, **declared)
    assert module.decode_query_rows <= seq.cache.q.size(2)
    new = [1] * len(lengths)
    new[0] = 2
    seq.feed(new)
    got = module.decode(seq.cache)
    assert got.shape == (len(lengths), 1, h, d) and got.dtype == dtype
    for b in range(len(lengths)):
        check(got[b, 0], *seq.want(b, w, d ** -0.5, pre=pre, w2=w2, post=post), what=f"slot {b}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("absent", ["pre", "post", "pre post", "conv", "conv pre", "conv post", "conv pre post"])
def test_mta_identity_stages(dtype, absent):
    h, d = 8, 64
    seq = Sequences([40, 130], h, h, d, dtype, 32, 10)
    w, w2 = conv_weight(h, 5, 7, dtype, seq.gen), None if "conv" in absent else conv_weight(h, 3, 3, dtype, seq.gen)
    pre, post = [None if name in absent.split() else head_weight(h, 4, dtype, seq.gen) for name in ("pre", "post")]
    module = mta_module(w, pre, w2, post, pre_head_identity=pre is None, pre_head_group=4, post_head_identity=post is None, post_head_group=4,
                        post_conv_identity=w2 is None)
    seq.feed([1, 1])
    got = module.decode(seq.cache)
    for b in range(2):
        check(got[b, 0], *seq.want(b, w, d ** -0.5, pre=pre, w2=w2, post=post), what=f"slot {b}")


@pytest.mark.parametrize("window", [1, 5, 64, 300])
@pytest.mark.parametrize("r2,s2", [(0, 0), (5, 7)])
def test_mta_window(window, r2, s2):
    h, d, dtype = 8, 64, torch.float32
    seq = Sequences([1, 20, 333, 700], h, 4, d, dtype, 16, 12)
    w, w2 = conv_weight(h, 6, 11, dtype, seq.gen), conv_weight(h, r2, s2, dtype, seq.gen) if r2 else None
    pre, post = head_weight(h, 4, dtype, seq.gen), head_weight(h, 4, dtype, seq.gen)
    module = mta_module(w, pre, w2, post, pre_head_group=4, post_head_group=4, post_conv_identity=not r2)
    seq.feed([1, 1, 1, 1])
    got = module.decode(seq.cache, window=window)
    for b in range(4):
        check(got[b, 0], *seq.want(b, w, d ** -0.5, pre=pre, w2=w2, post=post, window=window), what=f"slot {b}")


def test_mta_long():
    h, d, dtype = 16, 128, torch.bfloat16
    seq = Sequences([5001, 2600], h, h, d, dtype, 64, 13, scatter=False)
    w, w2 = conv_weight(h, 7, 7, dtype, seq.gen), conv_weight(h, 7, 7, dtype, seq.gen)
    pre, post = head_weight(h, h, dtype, seq.gen), head_weight(h, h, dtype, seq.gen)
    got = mta_module(w, pre, w2, post).decode(seq.cache)
    for b in range(2):
        check(got[b, 0], *seq.want(b, w, d ** -0.5, pre=pre, w2=w2, post=post), what=f"slot {b}")


@pytest.mark.parametrize("h,r2,s2,group", [(8, 3, 3, 0), (6, 2, 5, 3), (5, 7, 7, 5), (9, 9, 4, 1), (12, 12, 11, 6), (4, 1, 16, 0), (4, 32, 2, 2), (2, 17, 63, 0), (7, 6, 1, 0)])
@pytest.mark.parametrize("length", [2, 256, 257, 300, 505, 512, 513, 700])
def test_mta_rows_of_few_keys(h, r2, s2, group, length):
    """Rows around the lengths at which the stages behind the scores are laid out in another way; heads that no four divide."""
    d, dtype = 64, torch.float32
    print(f"mta decode h={h} {r2}x{s2} group={group} {length}", flush=True)
    seq = Sequences([length - 1, length // 2, 0], h, h, d, dtype, 32, r2 + 1, scatter=False)
    w, w2 = conv_weight(h, 2, 3, dtype, seq.gen), conv_weight(h, r2, s2, dtype, seq.gen)
    pre, post = head_weight(h, group or h, dtype, seq.gen), head_weight(h, group or h, dtype, seq.gen)
    plain = mta_module(w, None, w2, None, pre_head_identity=True, post_head_identity=True)
    full = mta_module(w, pre, w2, post, **(dict(pre_head_group=group, post_head_group=group) if group else {}))
    seq.feed([1, 1, 0])
    got, got2 = plain.decode(seq.cache), full.decode(seq.cache)
    for b in range(2):
        check(got[b, 0], *seq.want(b, w, d ** -0.5, w2=w2), what=f"slot {b}")
        check(got2[b, 0], *seq.want(b, w, d ** -0.5, pre=pre, w2=w2, post=post), what=f"slot {b}")
    assert not got[2].any() and not got2[2].any()
    for window in (3, 400):
        got2 = full.decode(seq.cache, window=window)
        for b in range(2):
            check(got2[b, 0], *seq.want(b, w, d ** -0.5, pre=pre, w2=w2, post=post, window=window), what=f"slot {b}, window {window}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_nothing_added_yet(dtype):
    """A new cache, one whose slots all sit the step out, one that was emptied: zeros."""
    seq = Sequences([0, 0], 4, 2, 64, dtype, 16, 8)
    w, w2 = conv_weight(4, 3, 3, dtype, seq.gen), conv_weight(4, 3, 3, dtype, seq.gen)
    pre = head_weight(4, 4, dtype, seq.gen)
    conv, full = conv_module(w), mta_module(w, pre, w2, pre)
    for counts in (None, [0, 0], [3, 5], [0, 0]):
        if counts:
            seq.cache.extend(counts) if not any(counts) else seq.feed(counts)
        got, got2 = conv.decode(seq.cache), full.decode(seq.cache)
        assert got.isfinite().all() and got2.isfinite().all() and got.any().item() == got2.any().item() == any(counts or [])
    for b in range(2):
        seq.cache.free(b)
    assert not conv.decode(seq.cache).any() and not full.decode(seq.cache).any()


def test_mta_weights_of_other_dtypes():
    h, d = 4, 64
    seq = Sequences([77], h, h, d, torch.float16, 16, 5)
    w, w2 = conv_weight(h, 3, 3, torch.float32, seq.gen), conv_weight(h, 3, 3, torch.float32, seq.gen)
    pre, post = head_weight(h, h, torch.float32, seq.gen), head_weight(h, h, torch.float32, seq.gen)
    module = mta_module(w, pre, w2, post)
    seq.feed([1])
    check(module.decode(seq.cache)[0, 0], *seq.want(0, w, d ** -0.5, pre=pre, w2=w2, post=post))
    module.wpsm_triton.to(torch.float16)
    check(module.decode(seq.cache)[0, 0], *seq.want(0, w, d ** -0.5, pre=pre.half(), w2=w2, post=post))


# ---- the module's own forward() ---------------------------------------------------------------------------------------------
def _close_to_forward(got, whole, bounds):
    """decode() is within `bounds` of the formulas, forward() in fp32 within what its own tests hold it to, rtol 1e-4 and atol 1e-5: so far apart they
    may be.  (A tap, a row or a head out of place is some hundredths.)"""
    got, whole = got.double().cpu(), whole.double().cpu()
    off = (got - whole).abs() - (bounds + 2 ** -24 * got.abs() + 1e-4 * whole.abs() + 1e-5)
    assert off.max() <= 0, f"{float((got - whole).abs().max())} apart, {float(off.max())} too far"


@pytest.mark.parametrize("r,s", [(3, 3), (6, 11), (3, 4), (2, 6), (1, 2)])
@pytest.mark.parametrize("n", [1, 5, 77, 300])
def test_conv_attention_is_the_last_row_of_forward(r, s, n):
    h, d, dtype = 4, 64, torch.float32
    seq = Sequences([n, n], h, h, d, dtype, 16, r, scatter=False)
    w = conv_weight(h, r, s, dtype, seq.gen)
    module = conv_module(w)
    with torch.no_grad():
        whole, _ = module(*(x[:, :, :n].contiguous().cuda() for x in (seq.q, seq.k, seq.v)), True, 0.2)
    got = module.decode(seq.cache, 0.2)
    _close_to_forward(got[:, :, 0], whole[:, :, -1], torch.stack([seq.want(b, w, 0.2)[1] for b in range(2)]))


@pytest.mark.parametrize("h,r,s,r2,s2,group,window", [(8, 3, 3, 3, 3, 0, 0), (8, 6, 11, 0, 0, 4, 0), (4, 5, 7, 2, 4, 2, 0), (4, 2, 4, 4, 6, 0, 0), (16, 3, 5, 5, 3, 0, 0),
                                                      (8, 6, 11, 0, 0, 2, 40), (4, 3, 4, 3, 5, 0, 100)])
@pytest.mark.parametrize("n", [1, 5, 77, 304])
def test_mta_is_the_last_row_of_forward(h, r, s, r2, s2, group, window, n):
    d, dtype = 64, torch.float32
    seq = Sequences([n, n], h, h, d, dtype, 16, r + max(r2, 3) - 1, scatter=False)
    w, w2 = conv_weight(h, r, s, dtype, seq.gen), conv_weight(h, r2, s2, dtype, seq.gen) if r2 else None
    pre, post = head_weight(h, group or h, dtype, seq.gen), head_weight(h, group or h, dtype, seq.gen)
    declared = dict(pre_head_group=group, post_head_group=group, post_conv_identity=not r2) if group else {}
    module = mta_module(w, pre, w2, post, **declared)
    mask = None
    if window:
        at = torch.arange(n, device="cuda")
        mask = ((at[None] <= at[:, None]) & (at[None] > at[:, None] - window)).expand(2, 1, n, n)
        module.use_mask = True
    with torch.no_grad():
        whole = module(*(x[:, :, :n].contiguous().cuda() for x in (seq.q, seq.k, seq.v)), mask, None)
    got = module.decode(seq.cache, window=window)
    bounds = torch.stack([seq.want(b, w, d ** -0.5, pre=pre, w2=w2, post=post, window=window)[1] for b in range(2)])
    _close_to_forward(got[:, 0], whole[:, -1], bounds)


# ---- a serving loop ------------------------------------------------------------------------------------------------------------
def test_prompt_then_tokens_then_fork_then_compact():
    """Prompts, a few steps, a beam that splits, one that ends, pages moved together, more steps: every step against whole sequences."""
    h, hkv, d, dtype = 4, 2, 64, torch.float32
    seq = Sequences([37, 64, 0, 3], h, hkv, d, dtype, 16, 6, n_pages=40, scatter=False)
    w = conv_weight(h, 4, 5, dtype, seq.gen)
    module = conv_module(w)

    def step(counts):
        seq.feed(counts)
        got = module.decode(seq.cache)
        for b, c in enumerate(counts):
            if c:
                check(got[b, :, 0], *seq.want(b, w, d ** -0.5), what=f"slot {b}")
            else:
                assert not got[b].any()

    step([1, 1, 0, 2])
    step([1, 0, 0, 1])
    seq.cache.fork(0, [2, 3])           # 3 held something else
    for x in (seq.q, seq.k, seq.v):
        x[2, :, :seq.cache.lengths[0]] = x[0, :, :seq.cache.lengths[0]]
        x[3, :, :seq.cache.lengths[0]] = x[0, :, :seq.cache.lengths[0]]
    assert seq.cache.lengths[2] == seq.cache.lengths[3] == 39
    step([1, 1, 1, 1])
    seq.cache.free(0)
    before = [seq.cache.pages_of(b) for b in range(4)]
    used = seq.cache.compact()
    assert sorted({p for b in range(4) for p in seq.cache.pages_of(b)}) == list(range(used)) and before != [seq.cache.pages_of(b) for b in range(4)]
    seq.cache.k[used:], seq.cache.v[used:] = float("nan"), float("nan")
    step([0, 1, 3, 1])
    step([5, 1, 1, 0])


def test_fork_between_extend_and_append():
    """Refused while the source's tokens are in no page; once appended - by a call or by a graph that the cache is told of - the copy has them."""
    h, d, dtype = 4, 64, torch.float32
    seq = Sequences([35, 3, 0], h, h, d, dtype, 16, 4, scatter=False)
    w = conv_weight(h, 4, 5, dtype, seq.gen)
    module = conv_module(w)
    n = 35

    def same(slot):
        for x in (seq.q, seq.k, seq.v):
            x[slot, :, :n] = x[0, :, :n]

    def new():
        return [x[:, :, n - 1:n].cuda() for x in (seq.q, seq.k, seq.v)]

    def step():
        seq.feed([1, 1, 1])
        got = module.decode(seq.cache)
        for b in range(3):
            check(got[b, :, 0], *seq.want(b, w, d ** -0.5), what=f"slot {b}")

    seq.cache.extend([1, 0, 0])
    n += 1
    with pytest.raises(RuntimeError, match="not been appended"):
        seq.cache.fork(0, 2)
    assert seq.cache.lengths == [36, 3, 0]
    seq.cache.append(*new())
    seq.cache.fork(0, 2)
    same(2)
    step()
    n += 1
    static = [x.clone() for x in new()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        seq.cache.append(*static)
    seq.cache.extend([1, 0, 0])
    n += 1
    for x, y in zip(static, new()):
        x.copy_(y)
    graph.replay()
    with pytest.raises(RuntimeError, match="not been appended"):
        seq.cache.fork(0, 1)
    seq.cache.mark_appended()
    seq.cache.fork(0, 1)
    same(1)
    step()


@pytest.mark.parametrize("n", [96, 100, 15])
def test_fork_of_a_new_prompt(n):
    """Samples of one prompt, straight after its append: whole pages are shared, one page is copied at most; all go on alone."""
    h, d, dtype, page = 4, 64, torch.bfloat16, 16
    seq = Sequences([n, 0, 0, 0], h, 2, d, dtype, page, 5, n_pages=n // page + 8, scatter=False)
    w = conv_weight(h, 5, 7, dtype, seq.gen)
    module = conv_module(w)
    free = seq.cache.free_pages
    seq.cache.fork(0, [1, 2, 3])
    assert all(seq.cache.pages_of(b)[:n // page] == seq.cache.pages_of(0)[:n // page] for b in range(4))
    assert seq.cache.free_pages == free - 3 * (n % page > 0)
    for x in (seq.q, seq.k, seq.v):
        x[1:, :, :n] = x[:1, :, :n]
    got = module.decode(seq.cache)
    check(got[0, :, 0], *seq.want(0, w, d ** -0.5))
    assert not got[1:].any()
    for _ in range(2):
        seq.feed([1, 1, 1, 1])
        got = module.decode(seq.cache)
        for b in range(4):
            check(got[b, :, 0], *seq.want(b, w, d ** -0.5), what=f"slot {b}")


def test_adopted_cache():
    h, d, dtype = 4, 64, torch.bfloat16
    seq = Sequences([50, 20], h, h, d, dtype, 16, 3, scatter=True)
    w = conv_weight(h, 3, 3, dtype, seq.gen)
    seq.feed([1, 1])
    c = seq.cache
    again = mta.PagedCache.adopt(c.k, c.v, c.q, c.table, c.lengths)
    assert torch.equal(conv_module(w).decode(again), conv_module(w).decode(c)) and again.free_pages == c.free_pages


def test_capture_and_replay():
    """A captured step follows the cache as it grows; eager work runs between the replays; two graphs hold their own workspaces."""
    h, d, dtype = 8, 64, torch.bfloat16
    seq = Sequences([30, 250], h, h, d, dtype, 16, 9, n_pages=64, max_pages=24, scatter=False)
    w, w2 = conv_weight(h, 5, 7, dtype, seq.gen), conv_weight(h, 3, 3, dtype, seq.gen)
    pre, post = head_weight(h, h, dtype, seq.gen), head_weight(h, h, dtype, seq.gen)
    first, second = conv_module(w), mta_module(w, pre, w2, post)
    xs = [torch.zeros(2, h, 1, d, dtype=dtype, device="cuda") for _ in range(3)]
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        seq.cache.extend(1)
        seq.cache.append(*xs)
        first.decode(seq.cache), second.decode(seq.cache)
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    with torch.cuda.graph(graphs[0]):
        seq.cache.append(*xs)
        outs.append(first.decode(seq.cache))
    with torch.cuda.graph(graphs[1]):
        outs.append(second.decode(seq.cache))
    with pytest.raises(RuntimeError, match="between replays"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            seq.cache.extend(1)
    for b, n in enumerate([30, 250]):
        for x in (seq.q, seq.k, seq.v):
            x[b, :, n] = 0                                   # (the zeros that were appended before the capture)
    for step in range(5):
        had = seq.cache.lengths
        seq.cache.extend([1, 1] if step != 2 else [0, 1])
        for x, whole in zip(xs, (seq.q, seq.k, seq.v)):
            x.copy_(torch.stack([whole[b, :, had[b]:had[b] + 1] for b in range(2)]))
        graphs[0].replay()
        graphs[1].replay()
        graphs[0].replay()                                   # (the same step again gives the same)
        torch.cuda.synchronize()
        eager = first.decode(seq.cache), second.decode(seq.cache)
        for b in range(2):
            if step == 2 and b == 0:
                assert not outs[0][b].any() and not outs[1][b].any()
                continue
            check(outs[0][b, :, 0], *seq.want(b, w, d ** -0.5), what=f"step {step} slot {b}")
            check(outs[1][b, 0], *seq.want(b, w, d ** -0.5, pre=pre, w2=w2, post=post), what=f"step {step} slot {b}")
        assert eager[0].shape == outs[0].shape and eager[1].shape == outs[1].shape


def test_on_another_stream():
    h, d, dtype = 4, 64, torch.float16
    seq = Sequences([300, 40], h, h, d, dtype, 16, 5, scatter=False)
    w, w2 = conv_weight(h, 3, 3, dtype, seq.gen), conv_weight(h, 3, 3, dtype, seq.gen)
    pre, post = head_weight(h, h, dtype, seq.gen), head_weight(h, h, dtype, seq.gen)
    module = mta_module(w, pre, w2, post)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for _ in range(3):
            seq.feed([1, 1])
            got = module.decode(seq.cache)
    stream.synchronize()
    for b in range(2):
        check(got[b, 0], *seq.want(b, w, d ** -0.5, pre=pre, w2=w2, post=post), what=f"slot {b}")


def test_two_calls_at_once():
    """Decodes of one cache on two streams, and of two caches, beside one another: each has its own workspace."""
    h, d, dtype = 8, 64, torch.bfloat16
    seqs = [Sequences([700, 90], h, h, d, dtype, 16, 7, seed=s, scatter=False) for s in (0, 1)]
    w, w2 = conv_weight(h, 5, 7, dtype, seqs[0].gen), conv_weight(h, 3, 3, dtype, seqs[0].gen)
    pre, post = head_weight(h, h, dtype, seqs[0].gen), head_weight(h, h, dtype, seqs[0].gen)
    conv, full = conv_module(w), mta_module(w, pre, w2, post)
    want = [(conv.decode(s.cache), full.decode(s.cache)) for s in seqs]
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    got = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 4]):
            s = seqs[i % 2].cache
            got.append((conv.decode(s), full.decode(s)))
    torch.cuda.synchronize()
    for i, (a, b) in enumerate(got):
        assert torch.equal(a, want[i % 2][0]) and torch.equal(b, want[i % 2][1])


def test_same_bits_every_time():
    h, d, dtype = 16, 128, torch.bfloat16
    seq = Sequences([3000, 700], h, h, d, dtype, 64, 11, scatter=False)
    w, w2 = conv_weight(h, 6, 11, dtype, seq.gen), conv_weight(h, 3, 3, dtype, seq.gen)
    pre, post = head_weight(h, h, dtype, seq.gen), head_weight(h, h, dtype, seq.gen)
    for module in (conv_module(w), mta_module(w, pre, w2, post)):
        first = module.decode(seq.cache)
        for _ in range(3):
            assert torch.equal(module.decode(seq.cache), first)


# ---- what is not a number, and what is not there --------------------------------------------------------------------------------
def _pair(dtype, lengths, seed=0, **more):
    h, d = 4, 64
    seq = Sequences(lengths, h, h, d, dtype, 16, 8, seed=seed, scatter=False, **more)
    w, w2 = conv_weight(h, 4, 5, dtype, seq.gen), conv_weight(h, 3, 3, dtype, seq.gen)
    pre, post = head_weight(h, h, dtype, seq.gen), head_weight(h, h, dtype, seq.gen)
    return seq, conv_module(w), mta_module(w, pre, w2, post), w, dict(pre=pre, w2=w2, post=post)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_not_finite(dtype, value):
    """A key, a value, a query that is not finite makes its own slot's results what the formulas make them, and no other's."""
    seq, conv, full, w, more = _pair(dtype, [50, 50, 50, 50])
    for b in range(4):
        seq.cache.free(b)
    seq.k[0, 1, 20, 3] = value
    seq.v[1, 1, 20, 3] = value
    seq.q[2, 1, 49, 3] = value
    seq.feed([50, 50, 50, 50])
    got, got2 = conv.decode(seq.cache), full.decode(seq.cache)
    for b in range(4):
        check(got[b, :, 0], *seq.want(b, w, 0.125), what=f"slot {b}")
        check(got2[b, 0], *seq.want(b, w, 0.125, **more), what=f"slot {b}")
    assert got[3].isfinite().all() and got2[3].isfinite().all() and not got[1].isfinite().all()


def test_large_scores():
    """Scores of some hundreds: one key takes all; the sum of exponentials does not overflow."""
    seq, conv, full, w, more = _pair(torch.float32, [120, 7])
    for b in range(2):
        seq.cache.free(b)
    seq.q *= 60
    seq.feed([120, 7])
    got, got2 = conv.decode(seq.cache), full.decode(seq.cache)
    for b in range(2):
        check(got[b, :, 0], *seq.want(b, w, 0.125))
        check(got2[b, 0], *seq.want(b, w, 0.125, **more))


def test_entries_that_are_no_pages():
    """A slot whose table names no page, or that holds more than it can, gets NaN; nothing is read through it; the others are as ever."""
    seq, conv, full, w, more = _pair(torch.bfloat16, [70, 70, 70, 70, 70])
    good = conv.decode(seq.cache), full.decode(seq.cache)
    seq.cache.table[0, 2] = seq.cache.k.size(0)
    seq.cache.table[1, 0] = -5
    seq.cache.state[0, 2] = 1 << 29
    seq.cache.state[0, 3] = -80
    got = conv.decode(seq.cache), full.decode(seq.cache)
    for x, y in zip(got, good):
        assert x[:4].isnan().all() and torch.equal(x[4], y[4])
    # ... and appending drops what has no page
    pools = seq.cache.k.clone(), seq.cache.v.clone()
    seq.cache.table.fill_(-1)
    seq.cache.append(*[torch.ones(5, 4, 70, 64, dtype=torch.bfloat16, device="cuda")] * 3)
    assert torch.equal(seq.cache.k.nan_to_num(7.0), pools[0].nan_to_num(7.0)) and torch.equal(seq.cache.v.nan_to_num(7.0), pools[1].nan_to_num(7.0))


def test_states_that_are_none():
    """Negative numbers and sums that pass 32 bits in a slot's state: NaN, also for slots that sit the step out; a long slot that sits it out is none of these."""
    seq, conv, full, w, more = _pair(torch.bfloat16, [70] * 7)
    for module in (conv, full):
        seq.cache._upload(everything=True)
        good = module.decode(seq.cache)
        for slot, (had, got) in enumerate(((70, -3), (-1, 0), (-70, -1), (2 ** 31 - 5, 10), (69, 2 ** 31 - 1), (70, 0))):
            seq.cache.state[0, slot], seq.cache.state[1, slot] = had, got
        out = module.decode(seq.cache)
        assert out[:5].isnan().all() and not out[5].any() and torch.equal(out[6], good[6])
    pools = [x.clone().nan_to_num(7.0) for x in (seq.cache.k, seq.cache.v, seq.cache.q)]
    seq.cache.state[1, 4], seq.cache.state[1, 6] = 0, 0
    seq.cache.append(*[torch.ones(7, 4, 70, 64, dtype=torch.bfloat16, device="cuda")] * 3)   # (what has no page is dropped)
    assert all(torch.equal(x.nan_to_num(7.0), y) for x, y in zip((seq.cache.k, seq.cache.v), pools))
    assert all(torch.equal(seq.cache.q[b].nan_to_num(7.0), pools[2][b]) for b in (0, 1, 2, 4, 5, 6))


def test_pools_beyond_32_bits():
    """Pages whose elements lie beyond 2**31, and bytes beyond 2**32."""
    h, d, page = 2, 128, 64
    pages = 2 ** 31 // (2 * page * d) + 40
    cache = mta.PagedCache(1, pages, h, d, page_size=page, max_pages=16, query_rows=4, dtype=torch.bfloat16)
    cache._free = list(range(pages - 12, pages))
    g = torch.Generator().manual_seed(3)
    q, k, v = [torch.randn(1, h, 500, d, generator=g).bfloat16() for _ in range(3)]
    cache.extend(500)
    cache.append(q.cuda(), k.cuda(), v.cuda())
    w = conv_weight(h, 4, 5, torch.bfloat16, g)
    check(conv_module(w).decode(cache)[0, :, 0], *token(q[0].double(), k[0].double(), v[0].double(), w.double(), d ** -0.5))
    ops.cache_copy_pages(cache.k, cache.v, [(pages - 12, 0), (pages - 11, pages - 1)])
    assert torch.equal(cache.k[0], cache.k[pages - 12]) and torch.equal(cache.v[pages - 1], cache.v[pages - 11])


# ---- the cache alone -------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["heads", "tokens", "odd", "fused"])
def test_append_layouts(dtype, layout):
    """Whatever the strides of the new tokens: the same rows arrive, bit for bit, and nothing else changes."""
    h, hkv, d, page, rows = 6, 3, 64, 16, 5
    g = torch.Generator().manual_seed(1)
    cache = mta.PagedCache(3, 30, h, d, hkv, page, 9, rows, dtype)
    for pool in (cache.k, cache.v, cache.q):
        pool.copy_(torch.randn(pool.shape, generator=g))
    want = [pool.cpu().clone() for pool in (cache.k, cache.v, cache.q)]
    for counts in ([20, 0, 3], [1, 1, 1], [40, 7, 0], [1, 0, 1]):
        had, n = cache.lengths, max(counts) + (layout == "heads")
        cache.extend(counts)
        x = [torch.randn(3, heads, n, d, generator=g).to(dtype) for heads in (h, hkv, hkv)]
        if layout == "heads":
            new = [t.cuda() for t in x]
        elif layout == "tokens":
            new = [t.transpose(1, 2).contiguous().cuda().transpose(1, 2) for t in x]
        elif layout == "odd":      # rows that are no whole vectors apart
            new = [torch.nn.functional.pad(t, (1, 2)).cuda()[..., 1:-2] for t in x]
        else:                      # one projection of all three
            new = list(torch.cat([t.transpose(1, 2) for t in x], 2).cuda().transpose(1, 2).split([h, hkv, hkv], 1))
        cache.append(*new)
        for b, c in enumerate(counts):
            for i in range(c):
                at = had[b] + i
                p = cache.pages_of(b)[at // page]
                want[0][p, :, at % page], want[1][p, :, at % page] = x[1][b, :, i], x[2][b, :, i]
                want[2][b, :, at % rows] = x[0][b, :, i]
        for pool, w in zip((cache.k, cache.v, cache.q), want):
            assert torch.equal(pool.cpu(), w)


@pytest.mark.parametrize("dtype,shape,n", [(torch.bfloat16, (700, 2, 16, 64), 600), (torch.float32, (9, 3, 16, 64), 1), (torch.float16, (64, 8, 64, 128), 40),
                                           (torch.float32, (6, 1, 1024, 128), 3)])
def test_copy_pages(dtype, shape, n):
    g = torch.Generator().manual_seed(2)
    k, v = [torch.randn(shape, generator=g).to(dtype) for _ in range(2)]
    order = torch.randperm(shape[0], generator=g).tolist()
    targets, sources = order[:n], order[n:]
    pairs = [(sources[i % len(sources)], t) for i, t in enumerate(targets)] + [(sources[0], sources[0])]
    dk, dv = k.cuda(), v.cuda()
    ops.cache_copy_pages(dk, dv, pairs)
    for s, t in pairs:
        k[t], v[t] = k[s], v[s]
    assert torch.equal(dk.cpu(), k) and torch.equal(dv.cpu(), v)
    ops.cache_copy_pages(dk, dv, torch.empty(0, 2, dtype=torch.int32))
    assert torch.equal(dk.cpu(), k)


def test_refusals_on_the_gpu():
    seq, conv, full, w, more = _pair(torch.bfloat16, [20, 20])
    c = seq.cache
    with pytest.raises(ValueError, match="newest 4 queries"):
        conv.decode(mta.PagedCache(2, 4, 4, 64, query_rows=3, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="newest 6 queries"):
        full.decode(mta.PagedCache(2, 4, 4, 64, query_rows=5, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="conv weight of 8 heads"):
        conv.decode(mta.PagedCache(2, 4, 8, 64, query_rows=4, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="window"):
        conv.decode(c, window=-1)
    with pytest.raises(ValueError, match="lives on cpu"):
        mta.TritonConvAttention(4, (4, 5)).to(torch.bfloat16).decode(c)
    x = torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="up to 20 tokens"):
        c.append(x, x, x)
    c.extend(1)
    with pytest.raises(TypeError):
        c.append(x.float(), x, x)
    with pytest.raises(ValueError, match="queries"):
        c.append(x[:1], x, x)
    with pytest.raises(ValueError, match="live on cpu"):
        c.append(x.cpu(), x, x)
    with pytest.raises(ValueError, match="contiguous"):
        ops.cache_copy_pages(c.k.transpose(1, 2), c.v.transpose(1, 2), [(0, 1)])
