"""Single-token attention over a paged cache, and what such a cache needs, as cases that can be timed.

A sequence lives in a slot; its keys and values lie in pages (page, key head, row, element) that a table per slot lists, its
newest queries in a ring (slot, head, position % rows, element).  A case is a dict of plain values:

    op       "conv" (fused conv-attention of the newest token), "mta" (Multi-Token Attention of the newest token), "append"
             (new tokens into pages and ring), "pages" (copies of pages, as a fork or a compaction makes them)
    dtype    of the cache, the weights and the results
    b h hkv  slots, query heads, key heads;  d  head size;  page  rows of a page
    length   tokens of the longest slot;  ragged: the others hold between an eighth and all of that
    new      tokens that a slot gets at most ("append");  pairs  pages to copy ("pages")
    r k      rows and keys of the (pre-softmax) conv kernel; r2, k2 of the post-softmax one, 0 = the identity tap, declared
    group    head weights block-diagonal with blocks of that many heads, declared; 0 = dense
    window   keys that a row sees at most, 0 = all
"""
from __future__ import annotations

import math
import random

import torch

own = False

_FIELDS = ("op", "dtype", "b", "h", "hkv", "d", "page", "length", "ragged", "new", "pairs", "r", "k", "r2", "k2", "group", "window")


def _case(name, *values):
    case = dict(zip(_FIELDS, values))
    return dict(case, name=name) if name else case


def listed():
    return [
        # one layer of a small model answering one user, a short context: launches and latency
        _case("conv_short_fp32", "conv", "float32", 1, 4, 4, 64, 16, 256, False, 0, 0, 3, 5, 0, 0, 0, 0),
        # a batch of chats of different lengths, keys shared by four heads
        _case("conv_chats_bf16", "conv", "bfloat16", 8, 32, 8, 128, 64, 4001, True, 0, 0, 6, 11, 0, 0, 0, 0),
        # one long document, a head size of 128, every head its own keys
        _case("conv_8k_bf16", "conv", "bfloat16", 1, 32, 32, 128, 64, 8192, False, 0, 0, 6, 11, 0, 0, 0, 0),
        # a full serving batch of long contexts
        _case("conv_batch_fp16", "conv", "float16", 16, 32, 32, 128, 128, 8192, True, 0, 0, 5, 7, 0, 0, 0, 0),
        # Multi-Token Attention, default kernel sizes, dense head weights, a short context
        _case("mta_short_bf16", "mta", "bfloat16", 1, 8, 8, 64, 16, 300, False, 0, 0, 3, 3, 3, 3, 0, 0),
        # two long contexts under a known weight structure: heads mixed in groups of 4, no conv behind the softmax
        _case("mta_4k_groups_bf16", "mta", "bfloat16", 2, 16, 16, 128, 64, 4096, False, 0, 0, 6, 11, 0, 0, 4, 0),
        # a serving batch of a trained layer: all four weights dense
        _case("mta_batch_dense_fp16", "mta", "float16", 16, 16, 16, 128, 64, 4096, True, 0, 0, 7, 7, 7, 7, 0, 0),
        # large kernels before and after the softmax, fp32, an odd number of tokens
        _case("mta_large_kernels_fp32", "mta", "float32", 4, 16, 16, 64, 32, 1001, True, 0, 0, 11, 15, 11, 15, 0, 0),
        # one token per chat goes into the cache, every step of every layer
        _case("append_step_bf16", "append", "bfloat16", 64, 32, 8, 128, 64, 4096, True, 1, 0, 6, 11, 0, 0, 0, 0),
        # prompts of a batch go into the cache at once
        _case("append_prompts_bf16", "append", "bfloat16", 4, 32, 32, 128, 64, 8192, True, 4096, 0, 6, 11, 0, 0, 0, 0),
        # a beam splits into eight: the page it is writing is copied for each
        _case("fork_8_bf16", "pages", "bfloat16", 8, 16, 16, 128, 64, 0, False, 0, 8, 0, 0, 0, 0, 0, 0),
        # what a burst of requests left scattered moves together
        _case("compact_1000_bf16", "pages", "bfloat16", 64, 32, 8, 128, 64, 0, False, 0, 1000, 0, 0, 0, 0, 0, 0),
    ]


_KERNELS = ((3, 3), (3, 5), (5, 5), (5, 7), (6, 11), (7, 7), (7, 9), (11, 15))


def _spread(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    """One more case of the ranges that the listed ones stand for."""
    most = {op: max(work(c)["bytes"] for c in listed() if c["op"] == op) for op in ("conv", "mta", "append", "pages")}
    while True:
        op = rng.choice(("conv", "conv", "conv", "mta", "mta", "mta", "append", "pages"))
        dtype = rng.choice(("bfloat16", "bfloat16", "float16", "float32"))
        h, d, page = rng.choice((4, 8, 12, 16, 32)), rng.choice((64, 128)), rng.choice((16, 32, 64, 128))
        hkv = h // rng.choice((1, 1, 2, 4))
        b = _spread(rng, 1, 64)
        length = _spread(rng, 1, 32768) if op != "pages" else 0
        r, k = rng.choice(_KERNELS)
        r2, k2, group, window = 0, 0, 0, 0
        if op in ("conv", "mta") and rng.random() < 0.25:
            window = _spread(rng, 1, 4096)
        if op == "mta":
            group = rng.choice((0, 0, 2, 4))
            if rng.random() < 0.6:
                r2, k2 = rng.choice(_KERNELS)
        new = _spread(rng, 1, length) if op == "append" else 0
        if op == "append" and rng.random() < 0.4:
            new = 1
        pairs = _spread(rng, 1, 1000) if op == "pages" else 0
        case = _case("", op, dtype, b, h, hkv, d, page, length, rng.random() < 0.6, new, pairs, r, k, r2, k2, group, window)
        if work(case)["bytes"] > most[op] or b * length * hkv * d > 2 ** 30:
            continue
        # (the plain form holds a product per tap)
        if op == "mta" and b * h * length * max(r2, 1) * r * k > 1.5e8 * (1 + (dtype != "float32")):
            continue
        return case


# ---- sizes that follow from a case ----------------------------------------------------------------------------------------
def _lengths(case):
    """Tokens of each slot, the new ones among them."""
    b, most = case["b"], case["length"]
    if not case["ragged"]:
        return [most] * b
    rng = random.Random(b * 1000003 + most)
    return [most if i == 0 else _spread(rng, max(1, most // 8), most) for i in range(b)]


def _added(case):
    """New tokens of each slot."""
    if case["op"] != "append":
        return [1] * case["b"]
    rng = random.Random(case["b"] * 1000003 + case["new"])
    return [min(n, case["new"] if not case["ragged"] or i == 0 else _spread(rng, max(1, case["new"] // 4), case["new"]))
            for i, n in enumerate(_lengths(case))]


def _rows(case):
    """Query rows whose raw scores the newest token needs."""
    return case["r"] + max(case["r2"], 1) - 1


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    b, h, hkv, d = case["b"], case["h"], case["hkv"], case["d"]
    if case["op"] == "pages":
        return {"bytes": case["pairs"] * hkv * case["page"] * d * size * 2 * 2, "flops": 0}
    if case["op"] == "append":
        ring = _rows(case)
        return {"bytes": sum((a * hkv * 2 + min(a, ring) * h) * d * size * 2 for a in _added(case)), "flops": 0}
    r2, group = max(case["r2"], 1), case["group"] or h
    seen = [min(n, case["window"]) if case["window"] else n for n in _lengths(case)]
    per_key = 2 * _rows(case) * d + 2 * r2 * case["r"] * case["k"] + 2 * d
    if case["op"] == "mta":
        per_key += 2 * r2 * group + 2 * group + 2 * case["r2"] * case["k2"]
    rows = b * h * d * (_rows(case) + 1)
    return {"bytes": (sum(seen) * hkv * d * 2 + rows) * size, "flops": sum(seen) * h * per_key}


# ---- inputs -----------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    """Pools, table and ring of a cache in use: pages in the order in which requests happened to take them."""
    dtype = getattr(torch, case["dtype"])
    b, h, hkv, d, page = case["b"], case["h"], case["hkv"], case["d"], case["page"]
    gen = torch.Generator("cuda").manual_seed(seed)
    cpu = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32 if dtype == torch.float32 else torch.float16).to(dtype)

    state = {"case": case}
    if case["op"] == "pages":
        n = case["pairs"]
        state["k"], state["v"] = normal(n + n // 2 + 1, hkv, page, d), normal(n + n // 2 + 1, hkv, page, d)
        order = torch.randperm(n + n // 2 + 1, generator=cpu).to(torch.int32)
        sources = order[n:][torch.randint(0, n // 2 + 1, (n,), generator=cpu)]   # a page may be copied to several places
        state["pairs"] = torch.stack([sources, order[:n]], 1).contiguous()
        return state
    lengths, added, ring = _lengths(case), _added(case), _rows(case)
    need = [-(-n // page) for n in lengths]
    # (some pages belong to nobody)
    order = torch.randperm(sum(need) + 3, generator=cpu).to(torch.int32)
    table = torch.full((b, max(need)), -1, dtype=torch.int32)
    at = 0
    for slot, n in enumerate(need):
        table[slot, :n] = order[at:at + n]
        at += n
    state["k"], state["v"] = normal(order.numel(), hkv, page, d), normal(order.numel(), hkv, page, d)
    state["q"] = normal(b, h, ring, d)
    state["table"] = table.cuda()
    state["lengths"] = torch.tensor(lengths, device="cuda")
    state["added"] = torch.tensor(added, device="cuda")
    if case["op"] == "append":
        # as a projection leaves them: token by token, all heads of a token together
        n = max(added)
        state["new"] = [normal(b, n, heads, d).transpose(1, 2) for heads in (h, hkv, hkv)]
    else:
        r2, k2 = max(case["r2"], 1), max(case["k2"], 1)
        state["w"] = _tap_and_noise(normal, h, case["r"], case["k"])
        state["w2"] = _tap_and_noise(normal, h, r2, k2) if case["r2"] else None
        blocks = torch.block_diag(*[torch.ones(case["group"] or h, case["group"] or h)] * (h // (case["group"] or h))).cuda()
        state["pre"], state["post"] = [((torch.eye(h, device="cuda") + 0.1 * normal(h, h).float()) * blocks).to(dtype) for _ in range(2)]
    if own:
        import multitokenatention_triton_amd as mta

        state["cache"] = mta.PagedCache.adopt(state["k"], state["v"], state["q"], table, lengths, added)
        if case["op"] == "conv":
            state["module"] = mta.TritonConvAttention(h, (case["r"], case["k"]), causal=True).to("cuda", dtype).requires_grad_(False)
            state["module"].weight.copy_(state["w"])
        elif case["op"] == "mta":
            sizes = (case["r2"], case["k2"]) if case["r2"] else (1, 1)
            config = mta.MTAConfig(query_kernel_size=case["r"], key_kernel_size=case["k"], after_sm_query_kernel_size=sizes[0], after_sm_key_kernel_size=sizes[1])
            module = mta.MTAAttentionTriton(h, config, dropout=0.0, causal=True).to("cuda", dtype).eval().requires_grad_(False)
            module.reset_mta_parameters()
            module.mta_conv_triton.weight.copy_(state["w"])
            if case["r2"]:
                module.mta_conv_after_sm_triton.weight.copy_(state["w2"])
            module.wpsm_triton.weight.copy_(state["pre"])
            module.wposm_triton.weight.copy_(state["post"])
            if case["group"]:
                module.declare_weight_structure(pre_head_group=case["group"], post_conv_identity=not case["r2"], post_head_group=case["group"])
            state["module"] = module
    return state


def _tap_and_noise(normal, h, r, k):
    """Conv kernels of a trained layer: about the pass-through tap they start from."""
    w = 0.1 * normal(h, r, k).float()
    w[:, r - 1, (k - 1) // 2] += 1.0
    return w.to(normal(1).dtype)


# ---- one pass ---------------------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        import multitokenatention_triton_amd as mta

        if case["op"] == "conv":
            return state["module"].decode(state["cache"], case["d"] ** -0.5, window=case["window"])
        if case["op"] == "mta":
            return state["module"].decode(state["cache"], window=case["window"])
        if case["op"] == "append":
            state["cache"].append(*state["new"])
            return state["k"], state["v"], state["q"]
        mta.ops.cache_copy_pages(state["k"], state["v"], state["pairs"])
        return state["k"], state["v"]
    if case["op"] == "pages":
        pairs = state["pairs"].to("cuda").long()
        for pool in (state["k"], state["v"]):
            pool[pairs[:, 1]] = pool[pairs[:, 0]]
        return state["k"], state["v"]
    if case["op"] == "append":
        return _append(state)
    return _decode(state)


def _keys(state, pool):
    """(B, Hkv, tokens, D) in 32 bits, out of the pages."""
    pages = pool[state["table"].clamp_min(0).long()]                  # (B, M, Hkv, page, D)
    return pages.permute(0, 2, 1, 3, 4).flatten(2, 3)[:, :, :state["case"]["length"]].float()


def _conv(x, w, rows):
    """sum over taps of w[h, r, t] x[b, h, j + r, key + t - (S-1)//2]: x (B, H, rows + R - 1, L) -> (B, H, rows, L)."""
    r, k = w.shape[1:]
    left = (k - 1) // 2
    x = torch.nn.functional.pad(x, (left, k - 1 - left)).unfold(2, r, 1).unfold(3, k, 1)
    return (x * w.float()[:, None, None]).sum((-2, -1))


def _decode(state):
    case = state["case"]
    b, h, hkv, d = case["b"], case["h"], case["hkv"], case["d"]
    mta_form, rows, n_raw = case["op"] == "mta", max(case["r2"], 1), _rows(case)
    k, v = _keys(state, state["k"]), _keys(state, state["v"])
    key = torch.arange(k.shape[2], device="cuda")
    at = state["lengths"][:, None] - n_raw + torch.arange(n_raw, device="cuda")          # positions of the query rows
    q = state["q"].gather(2, (at % n_raw)[:, None, :, None].expand(b, h, n_raw, d)).float()
    seen = (key <= at[..., None]) & (at[..., None] >= 0)
    if case["window"]:
        seen = seen & (key > at[..., None] - case["window"])
    seen = seen[:, None]                                                                 # (B, 1, rows, L)
    raw = torch.matmul(q.view(b, hkv, -1, d), k.transpose(2, 3)).view(b, h, n_raw, -1) * d ** -0.5
    s = _conv(torch.where(seen, raw, 0.0), state["w"], rows)
    seen = seen[:, :, -rows:]
    if mta_form:
        s = torch.matmul(state["pre"].float(), s.flatten(2)).view(s.shape)
    s = torch.where(seen, s, -math.inf)
    p = torch.where(seen, torch.exp(s - s.amax(-1, keepdim=True)), 0.0)
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-37)
    if mta_form:
        if case["r2"]:
            p = torch.where(seen[:, :, -1:], _conv(p, state["w2"], 1), 0.0)
        p = torch.matmul(state["post"].float(), p.flatten(2)).view(p.shape)
    o = torch.matmul(p.view(b, hkv, h // hkv, -1), v).view(b, h, 1, d)
    return (o.transpose(1, 2) if mta_form else o).to(state["k"].dtype)


def _append(state):
    case = state["case"]
    page, ring = case["page"], _rows(case)
    xq, xk, xv = state["new"]
    added, start = state["added"][:, None], (state["lengths"] - state["added"])[:, None]
    # (rows that a slot does not have write its last one again)
    i = torch.minimum(torch.arange(xk.shape[2], device="cuda"), added - 1)
    at = start + i
    pages = state["table"].gather(1, at // page).long()
    for pool, x in ((state["k"], xk), (state["v"], xv)):
        rows = x.transpose(1, 2).gather(1, i[:, :, None, None].expand(-1, -1, x.shape[1], x.shape[3]))
        pool[pages, :, at % page] = rows
    j = added - ring + torch.arange(ring, device="cuda")                                 # the newest queries
    at, old = (start + j) % ring, state["q"]
    index = at[:, None, :, None].expand(-1, xq.shape[1], -1, xq.shape[3])
    fresh = xq.gather(2, j.clamp_min(0)[:, None, :, None].expand_as(index))
    old.scatter_(2, index, torch.where((j >= 0)[:, None, :, None], fresh, old.gather(2, index)))
    return state["k"], state["v"], state["q"]


# ---- the definition, in 64 bits -----------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] in ("append", "pages"):
        return None      # (rows and pages as they are: nothing is computed)
    state = prepare(case, seed)
    return torch.stack([_token(case, state, b) for b in range(case["b"])])


def _token(case, state, b):
    """One slot's newest token, head by head and tap by tap."""
    h, share, page, window = case["h"], case["h"] // case["hkv"], case["page"], case["window"]
    n, n_raw, rows = _lengths(case)[b], _rows(case), max(case["r2"], 1)
    which = state["table"][b, :-(-n // page)].long()
    k, v = [torch.cat(list(pool[which].double().unbind(0)), 1)[:, :n] for pool in (state["k"], state["v"])]
    first = n - n_raw

    def visible(position):
        keep = torch.zeros(n, dtype=torch.bool, device="cuda")
        if position >= 0:
            keep[max(0, position - window + 1) if window else 0:position + 1] = True
        return keep

    def taps(x, w, out_rows):
        r, t = w.shape
        y = torch.zeros(out_rows, n, dtype=torch.float64, device="cuda")
        for dr in range(r):
            for dt in range(t):
                off = dt - (t - 1) // 2
                lo, hi = max(0, -off), min(n, n - off)
                if lo < hi:
                    y[:, lo:hi] += w[dr, dt] * x[dr:dr + out_rows, lo + off:hi + off]
        return y

    keep = torch.stack([visible(first + i) for i in range(n_raw)])
    scores = []
    for head in range(h):
        q = torch.stack([state["q"][b, head, (first + i) % n_raw] for i in range(n_raw)]).double()
        raw = torch.where(keep, (q @ k[head // share].T) / math.sqrt(case["d"]), 0.0)
        scores.append(taps(raw, state["w"][head].double(), rows))
    s = torch.stack(scores)                                                               # (H, rows, n)
    if case["op"] == "mta":
        s = torch.tensordot(state["pre"].double(), s, 1)
    p = torch.softmax(s.masked_fill(~keep[-rows:], -math.inf), -1).nan_to_num(0.0)        # (rows ahead of the first token: nothing)
    if case["op"] == "mta":
        if case["r2"]:
            p = torch.stack([taps(p[head], state["w2"][head].double(), 1) for head in range(h)]).masked_fill(~keep[-1], 0.0)
        p = torch.tensordot(state["post"].double(), p, 1)
        return torch.stack([p[head, 0] @ v[head // share] for head in range(h)])[None]
    return torch.stack([p[head] @ v[head // share] for head in range(h)])
