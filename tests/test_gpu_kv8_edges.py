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
