"""The paged KV cache without a GPU: what the entry points and the cache class refuse, workspaces, shared memory."""
import ctypes
import random
import types

import pytest
import torch

from shadowkv_amd import _lib
from shadowkv_amd.kernels import shadowkv
from shadowkv_amd.models.attention import Cache2Attn, PagedAttention
from shadowkv_amd.models.kvcache import PagedKVCache, method2kvcache

P = 4096  # an aligned address that nothing reads: every call here is refused before a launch
BF16 = torch.bfloat16


def _refused(name, args, text, **changed):
    given = dict(args, **changed)
    p = [ctypes.c_void_p(x) if k in PTRS else x for k, x in given.items()]
    rc = getattr(_lib.lib(), name)(*p, None)
    assert rc in (1, 2) and text in _lib.last_error(), (rc, _lib.last_error(), changed)


PTRS = {"lengths", "counts", "keep", "table", "held", "free", "left", "cu", "totals", "slots", "q", "k", "v", "kp", "vp",
        "out", "ws"}
RESERVE = dict(lengths=P, counts=P, table=P, stride=8, width=8, held=P, free=P, cap=9, left=P, B=2, rows=4, page=16, cu=P,
               totals=P, slots=P)
RELEASE = dict(lengths=P, keep=P, table=P, stride=8, width=8, held=P, free=P, cap=9, left=P, B=2, page=16)
WRITE = dict(k=P, kt=128, kh=128, v=P, vt=128, vh=128, kp=P, vp=P, sp=2048, sh=2048, ss=128, slots=P, rows=3, heads=1,
             pages=4, page=16)
PAGED = dict(q=P, qt=128, qh=128, kp=P, vp=P, sp=2048, sh=2048, ss=128, pages=4, page=16, table=P, stride=8, width=8,
             lengths=P, cu=P, rows=3, B=2, Hq=1, H=1, max_new=2, scale=0.1, window=0, out=P, ws=None, nbytes=0)
PACKED = dict(q=P, qt=128, qh=128, k=P, kt=128, kh=128, v=P, vt=128, vh=128, cu=P, rows=3, B=2, Hq=1, H=1, scale=0.1,
              window=0, out=P, ws=None, nbytes=0)


def test_entry_points_refuse():
    for name, args, pointers in (
            ("skv_paged_reserve", RESERVE, "lengths counts table held free left cu totals slots"),
            ("skv_paged_release", RELEASE, "lengths keep table held free left"),
            ("skv_paged_write", WRITE, "k v kp vp slots"), ("skv_paged_attn", PAGED, "q kp vp table lengths out"),
            ("skv_packed_attn", PACKED, "q k v cu out")):
        for p in pointers.split():
            _refused(name, args, "null pointer", **{p: None})
        if "page" in args:
            for page in (0, -16, 8, 24, 512):
                _refused(name, args, f"page={page}", page=page)
        for size in ("B", "width", "cap", "rows", "heads", "pages", "Hq", "H", "max_new"):
            if size in args:
                for value in (-1, 0) if not (name == "skv_paged_reserve" and size == "rows") else (-1,):
                    _refused(name, args, f"={value}", **{size: value})
    for name, args in (("skv_paged_reserve", RESERVE), ("skv_paged_release", RELEASE), ("skv_paged_attn", PAGED)):
        _refused(name, args, "width=", width=(1 << 26) + 1, stride=1 << 27)
    for name, args in (("skv_paged_reserve", RESERVE), ("skv_paged_release", RELEASE)):
        _refused(name, args, "stride 7", stride=7)
        _refused(name, args, "free=", cap=(1 << 30) + 1)
    _refused("skv_paged_reserve", RESERVE, "rows=", rows=(1 << 30) + 1)
    for p in ("k", "v", "kp", "vp"):
        _refused("skv_paged_write", WRITE, "aligned", **{p: P + 8})
    for s in ("kt", "kh", "vt", "vh", "sp", "sh", "ss"):
        _refused("skv_paged_write", WRITE, "aligned", **{s: 132})
    _refused("skv_paged_write", WRITE, "rows=", rows=1 << 28, heads=8)
    _refused("skv_paged_write", WRITE, "pages=", pages=(1 << 27) + 1)
    for name, args, pointers, strides in (("skv_paged_attn", PAGED, "q kp vp out", "qt qh sp sh ss"),
                                          ("skv_packed_attn", PACKED, "q k v out", "qt qh kt kh vt vh")):
        for p in pointers.split():
            _refused(name, args, "aligned", **{p: P + 8})
        for s in strides.split():
            _refused(name, args, "aligned", **{s: 132})
        _refused(name, args, "q_heads=3", Hq=3, H=2)
        _refused(name, args, "window=-1", window=-1)
        for scale in (float("inf"), float("nan")):
            _refused(name, args, "scale=", scale=scale)
        _refused(name, args, "rows=", rows=1 << 25, Hq=32)
    _refused("skv_paged_attn", PAGED, "rows=3", cu=None)
    _refused("skv_paged_attn", PAGED, "apart", ss=(1 << 24) + 8)
    _refused("skv_packed_attn", PACKED, "apart", kt=(1 << 24) + 8)
    _refused("skv_packed_attn", PACKED, "apart", vt=-8)


def test_workspaces():
    """None where one launch does; else enough for every share that the device may plan; 0 for bad sizes; a call with less
    is refused."""
    paged, packed = (getattr(_lib.lib(), f"skv_{x}_attn_workspace_bytes") for x in ("paged", "packed"))
    assert paged(1, 1, 32, 8, 1, 12, 64, 0) == 0
    assert paged(1, 1, 32, 8, 1, 4096, 64, 500) == 0
    assert packed(500, 3, 32, 8, 0) == 0
    assert packed(100000, 8, 32, 8, 0) == 0
    for need, name, args in ((paged(16, 16, 32, 8, 1, 2048, 64, 0), "skv_paged_attn",
                              dict(PAGED, rows=16, B=16, Hq=32, H=8, max_new=1, width=2048, page=64)),
                             (paged(90, 2, 8, 2, 90, 64, 64, 0), "skv_paged_attn",
                              dict(PAGED, rows=90, B=2, Hq=8, H=2, max_new=90, width=64, page=64)),
                             (packed(1100, 1, 1, 1, 0), "skv_packed_attn", dict(PACKED, rows=1100, B=1))):
        assert need > 0 and need % (130 * 4) == 0
        _refused(name, args, "workspace")
        _refused(name, args, "workspace", ws=P, nbytes=need - 1)
        _refused(name, args, "workspace", ws=P + 4, nbytes=need)
    for bad in ((0, 1, 1, 1, 1, 1, 16, 0), (1, 0, 1, 1, 1, 1, 16, 0), (1, 1, 3, 2, 1, 1, 16, 0), (1, 1, 1, 1, 0, 1, 16, 0),
                (1, 1, 1, 1, 1, 0, 16, 0), (1, 1, 1, 1, 1, 1, 16, -1), (1 << 30, 1, 1, 1, 1, 1, 16, 0)):
        assert paged(*bad) == 0
    for bad in ((0, 1, 1, 1, 0), (1, 0, 1, 1, 0), (1, 1, 3, 2, 0), (1, 1, 1, 1, -1)):
        assert packed(*bad) == 0


def test_host_tensors_and_wrong_ones_are_refused():
    ints = torch.zeros(2, dtype=torch.int32)
    table = torch.zeros(2, 4, dtype=torch.int32)
    pages, rows = torch.zeros(4, 1, 16, 128, dtype=BF16), torch.zeros(2, 1, 128, dtype=BF16)
    for call in (lambda: shadowkv.paged_reserve(ints, ints, table, ints, ints, ints[:1], rows=2, page=16),
                 lambda: shadowkv.paged_release(ints, ints, table, ints, ints, ints[:1], page=16),
                 lambda: shadowkv.paged_write(rows, rows, pages, pages.clone(), ints),
                 lambda: shadowkv.paged_attn(rows, pages, pages, table, ints),
                 lambda: shadowkv.packed_attn(rows, rows, rows, ints)):
        with pytest.raises(ValueError, match="device"):
            call()


def test_layouts_of_pages():
    """Which layouts are taken, and which share memory."""
    layout = shadowkv._pages_layout
    x = torch.empty(5, 2, 16, 128, dtype=BF16)
    assert layout(x.shape, x.stride())[:2] == ((5, 2, 16), (4096, 2048, 128))
    y = torch.empty(5, 16, 2, 128, dtype=BF16).transpose(1, 2)
    assert layout(y.shape, y.stride())[1] == (4096, 128, 256)
    assert layout(x[:, :1].expand(5, 2, 16, 128).shape, x[:, :1].expand(5, 2, 16, 128).stride())[2] is None
    for bad in (x[:, :, :12], torch.empty(5, 2, 24, 128), torch.empty(5, 2, 16, 64), torch.empty(5, 2, 16, 256)[..., ::2],
                torch.empty(2, 16, 128), torch.empty(0, 2, 16, 128), torch.empty(5, 2, 16, 132)[..., :128],
                torch.empty(1, device="meta").expand(2 ** 27 + 1, 1, 16, 128)):
        with pytest.raises(ValueError):
            layout(bad.shape, bad.stride())
    for pair in (torch.empty(5, 2, 2, 16, 128), torch.empty(5, 2, 16, 2, 128).permute(0, 3, 1, 2, 4)):
        k, v = pair[:, 0], pair[:, 1]
        dims = layout(k.shape, k.stride())[2]
        assert not shadowkv._pages_meet(dims, 2 * (v.storage_offset() - k.storage_offset()))
        assert shadowkv._pages_meet(dims, 0) and shadowkv._pages_meet(dims, 16)


def test_pages_that_share_memory_against_sets_of_bytes():
    rng = random.Random(2)
    seen = {True: 0, False: 0}
    for _ in range(200):
        shape, strides, extent = (rng.randint(1, 3), rng.randint(1, 3), 16, 128), [0, 0, 0, 1], 128
        for axis in rng.sample(range(3), 3):
            strides[axis] = extent + 8 * rng.choice([0, 16, 40, 41])
            extent = strides[axis] * (shape[axis] - 1) + extent
        dims = shadowkv._pages_layout(shape, tuple(strides))[2]
        at = [sum(i * s for i, s in zip((a, b, c), strides)) for a in range(shape[0]) for b in range(shape[1])
              for c in range(16)]
        d = 8 * rng.randint(-extent // 8 - 5, extent // 8 + 5)
        mine = {x for a in at for x in range(a, a + 128, 8)}
        want = any(x + d in mine for x in mine)
        assert shadowkv._pages_meet(dims, 2 * d) == want
        seen[want] += 1
    assert min(seen.values()) > 20


def _config(heads=8, kv_heads=2, head_dim=128, layers=3):
    return types.SimpleNamespace(num_attention_heads=heads, num_key_value_heads=kv_heads, hidden_size=heads * head_dim,
                                 num_hidden_layers=layers)


def test_cache_class():
    assert method2kvcache["paged"] is PagedKVCache and Cache2Attn[PagedKVCache] is PagedAttention
    cache = PagedKVCache(_config(), batch_size=3, max_length=100, device="cpu", page=16, pages=9)
    assert cache.k_pages.shape == (3, 9, 2, 16, 128) and cache.table.shape == (3, 7)
    assert cache.free_pages.tolist() == list(range(8, -1, -1)) and cache.free_count.item() == 9
    assert not cache.refused().any()
    assert PagedKVCache(_config(), batch_size=3, max_length=100, device="cpu").pages == 6
    cache.advance(100)
    rows = torch.zeros(3, 2, 1, 128, dtype=BF16)
    with pytest.raises(RuntimeError, match="capacity"):
        cache.update_kv_cache(rows, rows, 0)
    cache.clear()
    for call, text in ((lambda: cache.update_kv_cache(rows, rows, 0), "device"),
                       (lambda: cache.update_kv_cache(rows[:2], rows[:2], 0), "must be"),
                       (lambda: cache.update_kv_cache(rows, rows, 0, cache.asked), "must be"),
                       (lambda: cache.update_kv_cache(rows[:1], rows[:1], 0, cache.asked[:2]), "counts"),
                       (lambda: cache.update_kv_cache(rows[:1], rows[:1], 0, cache.asked, 0), "max_new"),
                       (lambda: cache.update_kv_cache(rows, rows, 1), "in a step of"),
                       (lambda: cache.attend(rows, 0), "in a step of"),
                       (lambda: cache.trim(cache.lengths.long(), 5), "int32"),
                       (lambda: cache.trim(cache.lengths, -1), "negative")):
        with pytest.raises(ValueError, match=text):
            call()
    assert cache.lengths.sum() == 0 and cache.incoming == 0 and cache.get_kv_len() == 0
    for wrong in (dict(page=48), dict(window=0), dict(max_length=0), dict(pages=0), dict(pages=2 ** 26),
                  dict(dtype=torch.float16), dict(config=_config(head_dim=64)), dict(max_length=2 ** 30 + 1)):
        with pytest.raises(ValueError):
            PagedKVCache(**{"config": _config(), "device": "cpu", "max_length": 64, "page": 64, **wrong})


@pytest.fixture
def cache(monkeypatch):
    """A cache whose kernels are lists."""
    from tests import paged_reference as ref

    def reserve(lengths, counts, table, held, free, count, *, rows, page):
        t, h, f = table.tolist(), held.tolist(), free[:count.item()].tolist()
        out = ref.reserve(lengths.tolist(), counts.tolist(), t, h, f, rows, page)
        for x, y in ((table, t), (held, h), (count, [len(f)])):
            x.copy_(torch.tensor(y))
        return [torch.tensor(x, dtype=torch.int32) for x in out]

    def release(lengths, keep, table, held, free, count, *, page):
        n, t, h, f = lengths.tolist(), table.tolist(), held.tolist(), free[:count.item()].tolist()
        ref.release(n, keep.tolist(), t, h, f, page)
        for x, y in ((lengths, n), (table, t), (held, h), (count, [len(f)]), (free[:len(f)], f)):
            x.copy_(torch.tensor(y))

    monkeypatch.setattr(shadowkv, "paged_reserve", reserve)
    monkeypatch.setattr(shadowkv, "paged_release", release)
    monkeypatch.setattr(shadowkv, "paged_write", lambda *a: None)
    return PagedKVCache(_config(), batch_size=2, max_length=100, device="cpu", page=16, pages=8)


def _step(cache, n, counts=None, layers=3, max_new=None):
    rows = torch.zeros(1 if counts is not None else 2, 2, n, 128, dtype=BF16)
    counts = None if counts is None else torch.tensor(counts, dtype=torch.int32)
    for layer in range(layers):
        cache.update_kv_cache(rows, rows, layer, counts, max_new)


def test_bookkeeping(cache):
    """Steps that end early, packed counts, refused sequences, dropped and ended ones, the capacity."""
    _step(cache, 20)
    assert cache.lengths.tolist() == [20, 20] and cache.get_kv_len() == 20 and cache.held.tolist() == [2, 2]
    _step(cache, 30, [25, 3], max_new=25)
    assert cache.lengths.tolist() == [45, 23] and cache.get_kv_len() == 45 and cache.cu.tolist() == [0, 25, 28]
    _step(cache, 10, layers=1)  # (held, though it went no further)
    assert cache.lengths.tolist() == [55, 33] and cache.get_kv_len() == 45 and cache.unfinished == 10
    with pytest.raises(RuntimeError, match="55 of 100"):
        cache.check_capacity(46)
    cache.trim(cache.start, 45)
    assert cache.lengths.tolist() == [45, 23] and cache.get_kv_len() == 45 and cache.unfinished == 0
    _step(cache, 55, [40, 15], max_new=40)  # 6 pages and 3: the second's are not free
    assert cache.refused().tolist() == [False, True]
    assert cache.lengths.tolist() == [85, 23] and cache.totals.tolist() == [85, 0] and cache.get_kv_len() == 85
    with pytest.raises(RuntimeError, match="capacity"):
        _step(cache, 16)
    cache.trim(torch.tensor([0, 100], dtype=torch.int32), 23)  # the first ends
    assert cache.held.tolist() == [0, 2] and cache.free_count.item() == 6 and cache.get_kv_len() == 23
    _step(cache, 15, [0, 15])
    assert not cache.refused().any() and cache.lengths.tolist() == [0, 38]
    _step(cache, 60, [30, 30], max_new=30)
    assert cache.lengths.tolist() == [30, 68] and cache.get_kv_len() == 68
    _step(cache, 5, [6, 0], max_new=6)  # (more than there are rows)
    assert cache.refused().tolist() == [True, False] and cache.lengths.tolist() == [30, 68]
    cache.clear()
    assert cache.free_count.item() == 8 and cache.table.eq(-1).all() and cache.get_kv_len() == 0


def test_more_new_tokens_than_the_host_said(cache):
    """Such a sequence is left as it is and known to refused(); the others' rows keep their places, and no length passes
    the host's bound."""
    _step(cache, 9, [4, 5], max_new=5)
    _step(cache, 12, [7, 5], max_new=5)
    assert cache.refused().tolist() == [True, False] and cache.totals.tolist() == [0, 10]
    assert cache.lengths.tolist() == [4, 10] and cache.held.tolist() == [1, 1] and cache.get_kv_len() == 10
    assert cache.cu.tolist() == [0, 7, 12] and cache.slots[:7].eq(-1).all() and cache.slots[7:].ge(0).all()
    assert cache.start.tolist() == [4, 5]
    cache.trim(cache.start, 5)
    assert cache.lengths.tolist() == [4, 5]
    _step(cache, 12, [7, 5], max_new=7)
    assert not cache.refused().any() and cache.lengths.tolist() == [11, 10] and cache.get_kv_len() == 12
    for _ in range(40):
        _step(cache, 2, [1, 1], max_new=1)
    _step(cache, 40, [1, 39], max_new=1)
    assert cache.lengths.tolist() == [52, 50] and int(cache.lengths.max()) <= cache.get_kv_len()


@pytest.mark.parametrize("name,args", [("skv_paged_attn", PAGED), ("skv_packed_attn", PACKED)])
def test_scales_that_pass_the_largest_number_are_refused(name, args):
    """As exponents of two: times log2(e)."""
    for scale in (2.4e38, -3.4e38):
        _refused(name, args, "scale=", scale=scale)
