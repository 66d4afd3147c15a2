"""The 8-bit KV cache without a GPU: what the entry points and the cache class refuse, and where they are found."""
import ctypes
import types

import pytest
import torch

from shadowkv_amd import _lib
from shadowkv_amd.kernels import shadowkv
from shadowkv_amd.models.attention import Cache2Attn, KV8Attention
from shadowkv_amd.models.kvcache import KV8Cache, method2kvcache

P = 4096  # an aligned address that nothing reads: every call here is refused before a launch


def _refused(name, args, text, **changed):
    lib = _lib.lib()
    given = dict(args, **changed)
    p = [ctypes.c_void_p(x) if k in PTRS else x for k, x in given.items()]
    rc = getattr(lib, name)(*p, None)
    assert rc in (1, 2) and text in _lib.last_error(), (rc, _lib.last_error(), changed)


PTRS = {"k", "v", "q", "k8", "v8", "ks", "vs", "start", "lengths", "counts", "codes", "scale", "ids", "out", "ws"}
WRITE = dict(k=P, ksb=128, ksh=128, kst=128, v=P, vsb=128, vsh=128, vst=128, k8=P, v8=P, csb=6400, csh=6400, css=128,
             ks=P, vs=P, ssb=4, ssh=4, start=P, counts=None, B=1, H=1, rows=1, cap=50, block=16)
READ = dict(codes=P, csb=6400, csh=6400, css=128, scale=P, ssb=4, ssh=4, ids=None, chunk=1, first=0, out=P, B=1, H=1,
            rows=4, cap=50, block=16)
ATTN = dict(q=P, qsb=128, qsh=128, qst=128, k8=P, v8=P, csb=6400, csh=6400, css=128, ks=P, vs=P, ssb=4, ssh=4,
            lengths=P, counts=None, B=1, Hq=1, H=1, rows=1, cap=50, block=16, softmax=0.1, window=0, sinks=0, out=P,
            ws=None, nbytes=0)


def test_entry_points_refuse():
    for p in ("k", "v", "k8", "v8", "ks", "vs", "start"):
        _refused("skv_kv8_write", WRITE, "null pointer", **{p: None})
    for p in ("q", "k8", "v8", "ks", "vs", "lengths", "out"):
        _refused("skv_kv8_attn", ATTN, "null pointer", **{p: None})
    for p in ("codes", "scale", "out"):
        _refused("skv_kv8_read", READ, "null pointer", **{p: None})
    for name, args in (("skv_kv8_write", WRITE), ("skv_kv8_read", READ), ("skv_kv8_attn", ATTN)):
        for block in (0, -16, 8, 48, 256):
            _refused(name, args, f"block={block}", block=block)
        for size in ("B", "H", "rows", "cap"):
            for value in (0, -1):
                _refused(name, args, f"{value}", **{size: value})
        _refused(name, args, "cap=", cap=(1 << 30) + 1)
        _refused(name, args, "aligned", css=136)
        _refused(name, args, "aligned", csh=6401)
        _refused(name, args, "batch=", B=1 << 29, rows=1)  # more threads than a launch has
        _refused(name, args, "batch=", rows=(1 << 30) + 1)
    for p in ("k", "v", "k8", "v8", "ks"):
        _refused("skv_kv8_write", WRITE, "aligned", **{p: P + 2})
    for stride in ("ksb", "ksh", "kst", "vsb", "vsh", "vst"):
        _refused("skv_kv8_write", WRITE, "aligned", **{stride: 129})
    _refused("skv_kv8_read", READ, "start=47", first=47)
    _refused("skv_kv8_read", READ, "start=-1", first=-1)
    _refused("skv_kv8_read", READ, "chunk=0", ids=P, chunk=0)
    _refused("skv_kv8_read", READ, "chunk=3", ids=P, chunk=3)
    _refused("skv_kv8_read", READ, "start=1", ids=P, chunk=2, first=1)
    for p in ("q", "k8", "out"):
        _refused("skv_kv8_attn", ATTN, "aligned", **{p: P + 8})
    for stride in ("qsb", "qsh", "qst"):
        _refused("skv_kv8_attn", ATTN, "aligned", **{stride: 132})
    _refused("skv_kv8_attn", ATTN, "q_heads=3", Hq=3, H=2)
    _refused("skv_kv8_attn", ATTN, "window=-1", window=-1)
    _refused("skv_kv8_attn", ATTN, "sinks=-1", sinks=-1)
    _refused("skv_kv8_attn", ATTN, "bytes apart", css=112)
    _refused("skv_kv8_attn", ATTN, "bytes apart", css=(1 << 24) + 16)
    _refused("skv_kv8_attn", ATTN, "workspace", cap=100000)


def test_workspace_sizes():
    """No workspace where one launch does; else partial rows of 130 floats that cover every chunk; 0 for bad sizes."""
    size = _lib.lib().skv_kv8_attn_workspace_bytes
    assert size(1, 32, 8, 1, 1000, 0, 0) == 0
    assert size(1, 32, 8, 1, 1 << 20, 500, 4) == 0
    assert size(1, 32, 8, 8192, 8192, 0, 0) == 0
    long = size(1, 32, 8, 1, 122880, 0, 0)
    assert long % (4 * 4 * 130) == 0 and long >= 2048 * 4 * 130 * 4
    need = size(2, 32, 8, 16, 4096, 0, 0)
    assert need > 0
    _refused("skv_kv8_attn", ATTN, "workspace", B=2, Hq=32, H=8, rows=16, cap=4096, ws=P, nbytes=need - 1)
    _refused("skv_kv8_attn", ATTN, "workspace", B=2, Hq=32, H=8, rows=16, cap=4096, ws=P + 4, nbytes=need)
    for bad in ((0, 32, 8, 1, 100, 0, 0), (1, 30, 8, 1, 100, 0, 0), (1, 32, 8, 0, 100, 0, 0), (1, 32, 8, 1, 0, 0, 0),
                (1, 32, 8, 1, 100, -1, 0), (1, 32, 8, 1, 100, 4, -1), (1, 32, 8, 1, (1 << 30) + 1, 0, 0)):
        assert size(*bad) == 0


def test_host_tensors_are_refused():
    k8 = torch.zeros(1, 2, 32, 128, dtype=torch.float8_e4m3fn)
    scale, at = torch.ones(1, 2, 2), torch.zeros(1, dtype=torch.int32)
    k = torch.zeros(1, 2, 1, 128, dtype=torch.bfloat16)
    for call in (lambda: shadowkv.kv8_write(k, k, k8, k8.clone(), scale, scale.clone(), at, block=16),
                 lambda: shadowkv.kv8_attn(k, k8, k8, scale, scale, at, block=16),
                 lambda: shadowkv.kv8_read(k8, scale, 0, 4, block=16),
                 lambda: shadowkv.kv8_read_chunks(k8, scale, torch.zeros(1, 2, 1, dtype=torch.int64), 8, block=16)):
        with pytest.raises(ValueError):
            call()


def _config(heads=8, kv_heads=2, head_dim=128, layers=2):
    return types.SimpleNamespace(num_attention_heads=heads, num_key_value_heads=kv_heads, hidden_size=heads * head_dim,
                                 num_hidden_layers=layers)


def test_cache_class():
    assert method2kvcache["kv8"] is KV8Cache and Cache2Attn[KV8Cache] is KV8Attention
    cache = KV8Cache(_config(), batch_size=3, max_length=100, device="cpu", block=32, window=64, sinks=4)
    assert cache.k8.shape == (2, 3, 2, 100, 128) and cache.k_scale.shape == (2, 3, 2, 4)
    assert cache.get_kv_len() == 0
    cache.advance(100)
    rows = torch.zeros(3, 2, 1, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="capacity"):
        cache.update_kv_cache(rows, rows, 0)
    assert cache.lengths.sum() == 0 and cache.get_kv_len() == 100  # (refused before anything changed)
    cache.clear()
    with pytest.raises(ValueError):
        cache.update_kv_cache(rows, rows, 0)  # (host tensors)
    assert cache.lengths.sum() == 0 and cache.incoming == 0 and cache.get_kv_len() == 0
    with pytest.raises(ValueError, match="in a step of"):
        cache.update_kv_cache(rows, rows, 1)
    with pytest.raises(ValueError, match="in a step of"):
        cache.attend(rows, 0)
    for wrong in (dict(block=48), dict(window=0), dict(sinks=3), dict(sinks=-1, window=4), dict(max_length=0),
                  dict(dtype=torch.float16), dict(config=_config(head_dim=64))):
        with pytest.raises(ValueError):
            KV8Cache(**{"config": _config(), "device": "cpu", "max_length": 64, **wrong})
