"""The paged cache's bookkeeping and what its entry points refuse, without a GPU."""
import ctypes

import pytest
import torch

import multitokenatention_triton_amd as mta
from multitokenatention_triton_amd import _lib, ops


def cache(**more):
    return mta.PagedCache(**{**dict(n_slots=3, n_pages=12, n_heads=4, head_dim=64, kv_heads=2, page_size=16, max_pages=5, query_rows=4, dtype=torch.float32,
                                    device="cpu"), **more})


def consistent(c):
    """Every page is free or counted once per slot that lists it; the device's table and state say what the host's lists say."""
    uses = [0] * c.k.size(0)
    for slot in range(c.n_slots):
        pages = c.pages_of(slot)
        assert len(pages) == -(-c.lengths[slot] // c.page_size) and c.table[slot, :len(pages)].tolist() == pages
        assert c.table[slot, len(pages):].eq(-1).all()
        for p in pages:
            uses[p] += 1
    assert uses == c._uses and sorted(c._free) == [p for p, u in enumerate(uses) if u == 0]
    assert (c.state[0] + c.state[1]).tolist() == c.lengths and c.state[1].tolist() == c._added


def test_extend_and_free():
    c = cache()
    consistent(c)
    assert c.longest == 1 and c.free_pages == 12
    c.extend([17, 0, 16])
    consistent(c)
    assert c.pages_of(0) == [0, 1] and c.pages_of(2) == [2] and c.lengths == [17, 0, 16] and c.longest == 17
    assert c.state.tolist() == [[0, 0, 0], [17, 0, 16]]
    c.extend(1)
    consistent(c)
    assert c.pages_of(1) == [3] and c.pages_of(2) == [2, 4] and c.state.tolist() == [[17, 0, 16], [1, 1, 1]]
    c.extend([0, 1, 0])
    assert c.state.tolist() == [[18, 1, 17], [0, 1, 0]]
    c.free(0)
    consistent(c)
    assert c.lengths == [0, 2, 17] and c.free_pages == 9
    c.extend([0, 15, 0])
    assert c.pages_of(1) == [3, 0]      # the lowest free page


def test_extend_refuses_and_changes_nothing():
    c = cache()
    c.extend([60, 60, 16])              # 4 + 4 + 1 pages
    for counts, error in (([21, 0, 0], RuntimeError), ([20, 20, 33], RuntimeError), ([-1, 0, 0], ValueError), ([1, 1], ValueError)):
        with pytest.raises(error):
            c.extend(counts)
        consistent(c)
        assert c.lengths == [60, 60, 16]
    c.extend([20, 20, 16])
    consistent(c)
    with pytest.raises(RuntimeError, match="0 free pages"):
        c.extend([0, 0, 1])


def test_fork_shares_whole_pages():
    c = cache()
    c.extend([31, 0, 40])
    c.extend([1, 0, 0])                 # two whole pages, the newest token in the second one
    with pytest.raises(RuntimeError, match="no CPU path"):
        c.fork(0, 1)                    # (the page with the newest token is copied)
    c = cache()
    c.extend([32, 0, 40])
    c.extend([0, 0, 0])
    c.fork(0, [1])
    consistent(c)
    assert c.pages_of(1) == c.pages_of(0) and c.lengths == [32, 32, 40] and c.free_pages == 7
    c.extend([1, 1, 0])
    consistent(c)
    assert c.pages_of(0)[:2] == c.pages_of(1)[:2] and c.pages_of(0)[2] != c.pages_of(1)[2]
    c.free(0)
    consistent(c)
    c.free(1)
    consistent(c)
    assert c.free_pages == 9
    c.fork(0, [2])                      # an empty slot empties its targets
    consistent(c)
    assert c.lengths == [0, 0, 0] and c.free_pages == 12
    for targets in (0, [1, 1], [3], [-1], ["1"]):
        with pytest.raises(ValueError):
            c.fork(0, targets)


def test_fork_waits_for_append():
    """Between extend and append a slot counts tokens that are in no page yet: a copy of it would never get them."""
    for counts in ([20, 0, 0], [32, 0, 0]):
        c = cache()
        c.extend([0, 40, 0])
        c.extend(counts)
        for targets in (1, [2], [1, 2]):
            with pytest.raises(RuntimeError, match=f"{counts[0]} tokens.*not been appended"):
                c.fork(0, targets)
            consistent(c)
            assert c.lengths == [counts[0], 40, 0] and c._added == counts
        c.fork(1, [])
        c.fork(2, [1])                  # (a slot that got none can be copied all the while)
        consistent(c)
        assert c.lengths == [counts[0], 0, 0]


def test_fork_of_a_new_prompt():
    """What has been appended is shared, however new it is."""
    c = cache(n_pages=4)
    c.extend([48, 0, 0])
    c.mark_appended()
    c.fork(0, [1, 2])                   # (copies would need six pages, one is free)
    consistent(c)
    assert c.pages_of(0) == c.pages_of(1) == c.pages_of(2) == [0, 1, 2] and c.free_pages == 1 and c.lengths == [48, 48, 48]
    assert c._added == [48, 0, 0]       # (the source's newest row can still be computed)
    x = torch.zeros(3, 4, 48, 64)
    with pytest.raises(RuntimeError, match="shared"):
        c.append(x, x[:, :2], x[:, :2])  # those tokens are the targets' as well now
    c.extend([0, 0, 1])
    consistent(c)
    assert c.pages_of(2) == [0, 1, 2, 3]
    with pytest.raises(RuntimeError, match="no CPU path"):
        c.append(x, x[:, :2], x[:, :2])


def test_mark_appended():
    """What a replayed graph appended, the cache is told of."""
    c = cache()
    c.extend([32, 0, 0])
    c.mark_appended()
    c.extend([0, 0, 0])
    c.fork(0, 1)
    consistent(c)
    c.extend([16, 0, 0])                # ... and that holds for one extend
    with pytest.raises(RuntimeError, match="not been appended"):
        c.fork(0, 2)
    c.free(0)
    c.fork(0, 2)
    assert c.lengths == [0, 32, 0]


def test_refused_fork_changes_nothing():
    """Pages that cannot be copied are found out before anything is released."""
    c = cache()
    c.extend([20, 30, 0])
    c.mark_appended()
    with pytest.raises(RuntimeError, match="no CPU path"):
        c.fork(0, [1, 2])
    consistent(c)
    assert c.lengths == [20, 30, 0] and c.pages_of(0) == [0, 1] and c.pages_of(1) == [2, 3] and c.state.tolist() == [[0, 0, 0], [20, 30, 0]]


def test_capture_is_looked_for_on_the_device_of_the_cache(monkeypatch):
    """Which stream is being captured is asked on the cache's own device, whatever the current one is."""
    current, capturing = ["cuda:0"], "cuda:1"

    class device:
        def __init__(self, d):
            self.d = str(d)

        def __enter__(self):
            current.append(self.d)

        def __exit__(self, *_):
            current.pop()

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: int(current[-1][-1]))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: current[-1] == capturing)

    class Pool:
        is_cuda = True

        def __init__(self, where, pool):
            self.device, self.size = torch.device(where), pool.size

    for where, longest in (("cuda:1", 80), ("cuda:0", 7), ("cuda:2", 7)):
        c = cache()
        c.extend([7, 0, 0])
        c.k = Pool(where, c.k)
        assert c.longest == longest
        if longest == 80:
            with pytest.raises(RuntimeError, match="between replays"):
                c.compact()
        else:
            assert c.compact() == 1


def test_compact_without_moves():
    c = cache()
    assert c.compact() == 0
    c.extend([16, 16, 16])
    assert c.compact() == 3
    c.free(2)
    assert c.compact() == 2
    c.free(0)
    with pytest.raises(RuntimeError, match="no CPU path"):
        c.compact()


def test_construction_refuses():
    for more in (dict(n_slots=0), dict(n_pages=0), dict(kv_heads=3), dict(head_dim=96), dict(page_size=48), dict(page_size=8), dict(page_size=2048),
                 dict(query_rows=0), dict(max_pages=0), dict(n_slots=70000), dict(n_slots=2.0)):
        with pytest.raises(ValueError):
            cache(**more)
    with pytest.raises(TypeError):
        cache(dtype=torch.float64)


def test_adopt():
    c = cache()
    c.extend([33, 16, 0])
    c.extend([1, 0, 0])
    again = mta.PagedCache.adopt(c.k, c.v, c.q, c.table, c.lengths, [1, 0, 0])
    consistent(again)
    assert again.lengths == c.lengths and again.state.tolist() == c.state.tolist() and again.free_pages == c.free_pages and again.k is c.k
    table = torch.tensor([[4, 5, 6], [4, 5, 7], [-1, -1, -1]])
    shared = mta.PagedCache.adopt(c.k, c.v, c.q, table, [40, 33, 0])
    consistent(shared)
    assert shared.free_pages == 8
    for tab, lengths, added in (([[4, 5, 6], [4, 5, 6], [0, 0, 0]], [40, 40, 0], None),      # a page that both write
                                ([[4, 5, 6], [4, 5, 7], [0, 0, 0]], [40, 33, 0], [20, 1, 0]),  # new tokens in a shared page
                                ([[4, 4, 6], [1, 2, 3], [0, 0, 0]], [40, 0, 0], None), ([[4, 12, 6], [1, 2, 3], [0, 0, 0]], [40, 0, 0], None),
                                ([[4, 5, 6], [1, 2, 3], [0, 0, 0]], [49, 0, 0], None), ([[4, 5, 6], [1, 2, 3], [0, 0, 0]], [40, 0, 0], [41, 0, 0]),
                                ([[4, 5, 6], [1, 2, 3]], [40, 0], None), ([[4, 5, 6], [1, 2, 3], [0, 0, 0]], [-1, 0, 0], None)):
        with pytest.raises(ValueError):
            mta.PagedCache.adopt(c.k, c.v, c.q, torch.tensor(tab), lengths, added)
    with pytest.raises(ValueError):
        mta.PagedCache.adopt(c.k, c.v.transpose(1, 2), c.q, table, [1, 1, 1])
    with pytest.raises(ValueError):
        mta.PagedCache.adopt(c.k, c.v, c.q[:, :3], table, [1, 1, 1])


def test_pairs_of_pages_that_are_refused():
    k = torch.zeros(6, 2, 16, 64)
    for pairs in ([(0, 6)], [(-1, 0)], [(0, 1), (2, 1)], [(0, 1), (1, 2)], [(0, 1), (3, 0)], torch.zeros(3), torch.zeros(2, 3, dtype=torch.int32),
                  torch.zeros(2, 2)):
        with pytest.raises(ValueError):
            ops.cache_copy_pages(k, k.clone(), pairs)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.cache_copy_pages(k, k.clone(), [(0, 1), (0, 2), (3, 3)])


def test_modules_refuse_without_a_gpu_and_where_they_cannot():
    c = cache()
    x = torch.zeros(3, 4, 1, 64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        c.append(x, x[:, :2], x[:, :2])
    with pytest.raises(RuntimeError, match="no CPU path"):
        mta.TritonConvAttention(4, (3, 3)).decode(c)
    config = mta.MTAConfig()
    with pytest.raises(RuntimeError, match="no CPU path"):
        mta.MTAAttentionTriton(4, config, 0.0, True).decode(c)
    with pytest.raises(ValueError, match="causal"):
        mta.MTAAttentionTriton(4, config, 0.0, False).decode(c)
    with pytest.raises(RuntimeError, match="dropout"):
        mta.MTAAttentionTriton(4, config, 0.1, True).decode(c)
    assert mta.MTAAttentionTriton(4, mta.MTAConfig(query_kernel_size=6, after_sm_query_kernel_size=3), 0.0, True).decode_query_rows == 8
    assert mta.TritonConvAttention(4, (6, 11)).decode_query_rows == 6


def test_abi_argument_codes():
    """Every refusal happens on the host, before anything is launched."""
    lib = _lib.load()
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    good = dict(k=p, v=p, q=p, table=p, state=p, n_pages=8, slots=2, max_pages=4, page=16, heads=4, kv_heads=2, head_dim=64, query_rows=8, dtype=0)

    def conv(longest=64, r=3, s=3, window=0, w=p, o=p, ws=p, size=1 << 40, wd=0, **more):
        c = _lib.Cache(**{**good, **more})
        return lib.mta_conv_attn_decode(ctypes.byref(c), w, o, ws, size, longest, r, s, window, 0.1, wd, None)

    def full(longest=64, r=3, s=3, r2=3, s2=3, g1=0, g2=0, window=0, w=p, pre=p, w2=p, post=p, o=p, ws=p, size=1 << 40, wd=0, **more):
        c = _lib.Cache(**{**good, **more})
        return lib.mta_decode(ctypes.byref(c), w, pre, w2, post, o, ws, size, longest, r, s, r2, s2, g1, g2, window, 0.1, wd, None)

    for call in (conv, full):
        for more, code in ((dict(k=None), -1), (dict(state=None), -1), (dict(w=None), -1), (dict(o=None), -1), (dict(dtype=3), -2), (dict(wd=7), -2), (dict(slots=0), -3),
                           (dict(n_pages=0), -3), (dict(page=24), -3), (dict(page=8), -3), (dict(page=2048), -3), (dict(longest=65), -3), (dict(longest=0), -3),
                           (dict(window=-1), -3), (dict(query_rows=2), -3), (dict(slots=70000), -3), (dict(r=33), -4), (dict(s=64), -4), (dict(r=0), -4), (dict(kv_heads=3), -5),
                           (dict(k=p + 4), -6), (dict(q=p + 8), -6), (dict(w=p + 2), -6), (dict(head_dim=96), -7), (dict(size=0, max_pages=64, longest=1024), -10)):
            assert call(**more) == code, (call.__name__, more)
    for more, code in ((dict(g1=3), -5), (dict(g2=-1), -5), (dict(w2=None), -1), (dict(ws=None), -1), (dict(r2=33), -4), (dict(s2=0), -4), (dict(r=6, r2=4), -3),
                       (dict(post=p + 2), -6), (dict(ws=p + 4), -6)):
        assert full(**more) == code, more
    c = _lib.Cache(**good)
    strides = (ctypes.c_int64 * 9)(*[64] * 9)
    odd = (ctypes.c_int64 * 9)(*[64] * 8, 66)
    assert lib.mta_cache_append(ctypes.byref(c), p, None, p, strides, 1, None) == -1
    assert lib.mta_cache_append(ctypes.byref(c), p, p, p, strides, 0, None) == -3
    assert lib.mta_cache_append(ctypes.byref(c), p, p, p, odd, 1, None) == -6
    assert lib.mta_cache_append(ctypes.byref(c), p, p, p + 4, strides, 1, None) == -6
    pairs = (ctypes.c_int32 * 4)(0, 1, 2, 8)
    assert lib.mta_cache_copy_pages(p, p, 8, 64, pairs, 2, None) == -3
    assert lib.mta_cache_copy_pages(p, None, 8, 64, pairs, 1, None) == -1
    assert lib.mta_cache_copy_pages(p, p, 8, 60, pairs, 1, None) == -6
    assert lib.mta_cache_copy_pages(p, p, 0, 64, pairs, 1, None) == -3
    assert lib.mta_cache_copy_pages(p, p, 8, 64, pairs, 0, None) == 0
    assert lib.mta_conv_attn_decode_workspace(ctypes.byref(c), 0, 3, 3, 0) == -3 and lib.mta_conv_attn_decode_workspace(ctypes.byref(c), 64, 3, 3, 0) >= 0
    assert lib.mta_decode_workspace(ctypes.byref(c), 64, 3, 3, 3, 3, 3, 0, 0) == -5 and lib.mta_decode_workspace(ctypes.byref(c), 64, 3, 3, 3, 3, 0, 0, 0) > 0


def test_workspaces_hold_whole_vectors():
    """Kernels read and write every part of a workspace 16 bytes at a time: it begins on 16 bytes, and so does each of its parts, whatever is odd.
    (The parts behind the rows' statistics end the workspace and are whole vectors themselves: its size shows where they begin.)"""
    lib = _lib.load()
    p = 1 << 20

    def made(slots, heads, keys):
        return _lib.Cache(k=p, v=p, q=p, table=p, state=p, n_pages=4096, slots=slots, max_pages=-(-keys // 64), page=64, heads=heads, kv_heads=heads, head_dim=64,
                          query_rows=32, dtype=0)

    for slots, heads, r2, keys in ((3, 5, 7, 200), (3, 5, 7, 700), (1, 1, 3, 200), (1, 1, 1, 1), (3, 3, 9, 2817), (5, 7, 5, 769), (2, 4, 4, 300)):
        c = made(slots, heads, keys)
        assert lib.mta_decode_workspace(ctypes.byref(c), keys, 3, 3, r2, 3, 0, 0, 0) % 16 == 0, (slots, heads, r2, keys)
    c = made(3, 5, 4096)
    size = lib.mta_conv_attn_decode_workspace(ctypes.byref(c), 4096, 3, 3, 0)
    assert size > 0
    for off, code in ((4, -6), (8, -6)):
        assert lib.mta_conv_attn_decode(ctypes.byref(c), p, p, p + off, size, 4096, 3, 3, 0, 0.1, 0, None) == code
        assert lib.mta_decode(ctypes.byref(c), p, p, p, p, p, p + off, 1 << 40, 4096, 3, 3, 3, 3, 0, 0, 0, 0.1, 0, None) == code


def test_longest_rows():
    """Multi-Token Attention's rows go as far as its launches do, and no size on the way wraps round; single-pass attention's go further."""
    lib = _lib.load()
    p = 1 << 20
    c = _lib.Cache(k=p, v=p, q=p, table=p, state=p, n_pages=1 << 20, slots=2, max_pages=1 << 20, page=1024, heads=4, kv_heads=4, head_dim=64, query_rows=64, dtype=0)
    most = 1 << 23
    for r2, s2 in ((1, 1), (3, 3), (32, 63)):
        size = lib.mta_decode_workspace(ctypes.byref(c), most, 3, 3, r2, s2, 0, 0, 0)
        assert size >= 4 * 2 * 4 * r2 * most
        assert lib.mta_decode_workspace(ctypes.byref(c), most + 1, 3, 3, r2, s2, 0, 0, 0) == -3
        assert lib.mta_decode(ctypes.byref(c), p, p, p, p, p, p, size, most + 1, 3, 3, r2, s2, 0, 0, 0, 0.1, 0, None) == -3
    assert lib.mta_conv_attn_decode_workspace(ctypes.byref(c), 1 << 30, 3, 3, 0) >= 0
    assert lib.mta_conv_attn_decode_workspace(ctypes.byref(c), (1 << 30) + 1, 3, 3, 0) == -3
