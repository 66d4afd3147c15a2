"""The 8-bit cache class's bookkeeping without a GPU: steps that end early, counts, dropped tokens, the capacity."""
import types

import pytest
import torch

from shadowkv_amd.kernels import shadowkv
from shadowkv_amd.models.kvcache import KV8Cache


@pytest.fixture
def cache(monkeypatch):
    monkeypatch.setattr(shadowkv, "kv8_write", lambda *a, **kw: None)
    config = types.SimpleNamespace(num_attention_heads=8, num_key_value_heads=2, hidden_size=1024, num_hidden_layers=3)
    return KV8Cache(config, batch_size=2, max_length=100, device="cpu")


def _rows(T):
    return torch.zeros(2, 2, T, 128, dtype=torch.bfloat16)


def _ints(*x):
    return torch.tensor(x, dtype=torch.int32)


def _step(cache, T, counts=None, layers=3):
    for layer in range(layers):
        cache.update_kv_cache(_rows(T), _rows(T), layer, counts)


def test_steps_that_end_before_the_last_layer_are_counted(cache):
    _step(cache, 40)
    assert cache.get_kv_len() == 40
    _step(cache, 30, layers=2)  # (its tokens are held: the device lengths went on at layer 0)
    assert cache.lengths.tolist() == [70, 70] and cache.get_kv_len() == 40
    with pytest.raises(RuntimeError, match="70 of 100 tokens held, 31 new"):
        cache.check_capacity(31)
    with pytest.raises(RuntimeError, match="capacity"):
        cache.update_kv_cache(_rows(31), _rows(31), 0)
    assert cache.lengths.tolist() == [70, 70]
    _step(cache, 30)
    assert cache.lengths.tolist() == [100, 100] and cache.get_kv_len() == 100
    with pytest.raises(RuntimeError, match="capacity"):
        cache.check_capacity(1)
    cache.clear()
    _step(cache, 60, layers=1)
    cache.clear()
    _step(cache, 100)
    assert cache.get_kv_len() == 100


def test_steps_that_are_advanced_by_hand(cache):
    for n in range(5):  # (the last layer is another cache's)
        _step(cache, 20, layers=2)
        cache.advance(20)
        assert cache.get_kv_len() == 20 * (n + 1) and cache.unfinished == 0
    with pytest.raises(RuntimeError, match="capacity"):
        cache.check_capacity(1)


def test_counts_of_later_layers(cache):
    cache.update_kv_cache(_rows(5), _rows(5), 0)
    with pytest.raises(ValueError, match="counts"):
        cache.update_kv_cache(_rows(5), _rows(5), 1, _ints(3, 5))
    cache.update_kv_cache(_rows(5), _rows(5), 1)
    cache.clear()
    _step(cache, 5, _ints(3, 5))
    assert cache.lengths.tolist() == [3, 5] and cache.get_kv_len() == 5


def test_trim(cache):
    _step(cache, 60, _ints(7, 50))
    cache.trim(cache.lengths, 50)  # (the padding of the prompts)
    assert cache.lengths.tolist() == [7, 50] and cache.get_kv_len() == 50
    for _ in range(12):  # five drafted tokens a step, one or two of them kept
        _step(cache, 5)
        cache.trim(cache.start + _ints(2, 1), cache.get_kv_len() - 4)
    assert cache.lengths.tolist() == [31, 62] and cache.get_kv_len() == 62
    with pytest.raises(ValueError, match="in a step of 0"):
        cache.update_kv_cache(_rows(5), _rows(5), 1)
    with pytest.raises(ValueError, match="in a step of 0"):
        cache.attend(_rows(5), 0)
    _step(cache, 9, layers=2)
    cache.trim(cache.start, 62)  # (a step that failed)
    assert cache.lengths.tolist() == [31, 62] and cache.get_kv_len() == 62
    cache.trim(_ints(-4, 1000), 100)
    assert cache.lengths.tolist() == [0, 62] and cache.get_kv_len() == 62
    cache.trim(cache.lengths, 10)
    assert cache.lengths.tolist() == [0, 10] and cache.get_kv_len() == 10
    for wrong in (_ints(1), _ints(1, 2).long(), _ints(1, 2).view(1, 2)):
        with pytest.raises(ValueError):
            cache.trim(wrong, 5)
    with pytest.raises(ValueError):
        cache.trim(cache.lengths, -1)


def test_windows_that_no_call_takes():
    config = types.SimpleNamespace(num_attention_heads=8, num_key_value_heads=2, hidden_size=1024, num_hidden_layers=1)
    for wrong in (dict(window=2 ** 31), dict(window=5, sinks=2 ** 31)):
        with pytest.raises(ValueError):
            KV8Cache(config, max_length=64, device="cpu", **wrong)
