"""The edges of the 8-bit cache's attention: what lies behind a sequence's end, padding, scores and scales of every size,
and the many-row form's own paths (large workgroups without shares, more workgroups than the chip holds at once)."""
import math

import pytest
import torch

from shadowkv_amd import _lib
from shadowkv_amd.kernels import shadowkv

from .test_gpu_kv8 import BF16, D, E4M3, _caches, _filled, _queries, _say, _see

pytestmark = pytest.mark.gpu


def _ints(x, gpu):
    return None if x is None else torch.tensor(x, dtype=torch.int32, device=gpu)


@pytest.mark.parametrize("H,G,T,cap", [(2, 4, 40, 70), (2, 4, 40, 129), (1, 4, 150, 331), (2, 4, 40, 2570),
                                       (2, 4, 40, 2627), (8, 4, 33, 8010)])
def test_attn_rows_behind_the_end(gpu, H, G, T, cap):
    """Caches whose capacity ends inside a tile, in a larger buffer: the same bits whether NaN or zeros lie behind the
    capacity (a NaN that reached the products would change the form that they take) and behind a shorter sequence."""
    _say(f"kv8_attn behind the end H={H} T={T} cap={cap}")
    g = torch.Generator().manual_seed(cap)
    q = _queries(2, H * G, T, g, gpu)
    whole = _filled(2, H, cap + 80, 16, g, gpu)
    caches = [c[:, :, :cap] for c in whole[:2]] + whole[2:]
    for lengths in ([cap, cap - 1], [cap - 3, T + 1]):
        got = []
        for code in (0x00, 0x7f):
            for c in whole[:2]:
                for b, n in enumerate(lengths):
                    c.view(torch.uint8)[b, :, n:] = code
            got.append(shadowkv.kv8_attn(q, *caches, _ints(lengths, gpu), block=16))
        assert not got[0].isnan().any() and torch.equal(*got), lengths


@pytest.mark.parametrize("H,G,T,cap", [(2, 4, 3, 128), (2, 4, 3, 2500), (2, 4, 6, 2500), (2, 4, 45, 128), (2, 4, 45, 2500),
                                       (1, 16, 40, 700), (8, 4, 33, 8000)])
def test_attn_padding_queries(gpu, H, G, T, cap):
    """Padding's queries may hold anything, one infinity and finite ones whose scores overflow among it: its rows are
    zeros, and the sequences' own rows have the bits that they have beside padding of zeros."""
    _say(f"kv8_attn padding queries H={H} G={G} T={T} cap={cap}")
    g = torch.Generator().manual_seed(T + cap)
    caches = _filled(3, H, cap, 32, g, gpu)
    lengths, counts = [min(cap, 2432), 64, cap // 64 * 64], [T - 1, 1, 0]
    q = _queries(3, H * G, T, g, gpu)
    pad = torch.zeros(3, T, dtype=torch.bool)
    for b, n in enumerate(counts):
        pad[b, n:] = True
    pad = pad.to(gpu)[:, None, :, None]
    one = torch.zeros(D, device=gpu)
    one[17] = 1.0
    call = lambda x: shadowkv.kv8_attn(x, *caches, _ints(lengths, gpu), _ints(counts, gpu), block=32)  # noqa: E731
    want = call(q.masked_fill(pad, 0.0))
    assert not want.isnan().any() and (want[pad[:, 0, :, 0]] == 0).all() and (want[0, 0] != 0).any()
    for odd in (math.nan, math.inf, -math.inf, 3e38, -3e38, torch.where(one > 0, math.inf, 0.5),
                torch.where(one > 0, -math.inf, -0.5), one * 3e38):
        x = torch.where(pad, torch.as_tensor(odd, device=gpu).to(BF16), q)
        assert torch.equal(call(x), want), odd
