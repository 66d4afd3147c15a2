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


@pytest.mark.parametrize("T,cap", [(1, 320), (6, 2500), (40, 320), (40, 2560), (300, 512)])
def test_attn_scores_past_32_bits_steps(gpu, T, cap):
    """Scores so large that neighbouring fp32 numbers differ by whole units, all equal: the mean of the values. Tolerance:
    the output's rounding, 2^-8 of the value, the fp32 sums', 2^-23 a key; and a score S (in units of log2) that is a
    product rounded to fp32 for one key and not for another moves a weight by up to 2^(2 S 2^-24), and the mean with it by
    that much, less 1, of the values' range, but never out of their range."""
    _say(f"kv8_attn large scores T={T} cap={cap}")
    g = torch.Generator().manual_seed(T)
    for size in (300.0, 3e4, 1.7e7, 3.1e9):
        for factor in (0.11, 0.0937, 0.087):
            k = torch.full((1, 2, cap, D), 13.0)
            v = torch.rand(1, 2, cap, D, generator=g) + 1.0
            caches = _caches(1, 2, cap, 32, g, gpu)
            shadowkv.kv8_write(k.to(BF16).to(gpu), v.to(BF16).to(gpu), *caches, _ints([0], gpu), block=32)
            vd = caches[1].cpu().double() * caches[3].cpu().double().repeat_interleave(32, 2)[:, :, :cap, None]
            q = torch.full((1, 8, T, D), size).to(BF16).to(gpu)
            got = shadowkv.kv8_attn(q, *caches, _ints([cap], gpu), block=32, scale=factor).cpu().double()
            want = vd.cumsum(2)[:, :, cap - T:] / torch.arange(cap - T + 1, cap + 1).view(1, 1, T, 1)
            want = want.repeat_interleave(4, 1).transpose(1, 2)
            score = abs(q[0, 0, 0, 0].item()) * 13 * D * factor / math.log(2)
            moved = min(1.0, math.expm1(min(1.0, 2 * score * 2.0 ** -24) * math.log(2))) * (vd.max() - vd.min())
            assert ((got - want).abs() <= want * (2.0 ** -8 + cap * 2.0 ** -23) + moved).all(), (size, factor)


@pytest.mark.parametrize("T,cap", [(1, 320), (1, 2500), (6, 320), (6, 2500), (40, 320), (40, 2500)])
def test_attn_scores_of_minus_infinity(gpu, T, cap):
    """A query all of whose scores are -inf divides zero by zero, as by the formula: NaN. One that sees nothing is
    zeros, and the others are what they are without it."""
    _say(f"kv8_attn scores of -inf T={T} cap={cap}")
    g = torch.Generator().manual_seed(T + cap)
    caches = _filled(2, 2, cap, 32, g, gpu)
    for c in caches[:2]:
        c[..., 3] = torch.ones((), device=gpu).to(E4M3)
    q = _queries(2, 8, T, g, gpu)
    q[..., 3] = 0.0
    at, n = _ints([256, T // 2], gpu), _ints([T, T], gpu)
    want = shadowkv.kv8_attn(q, *caches, at, n, block=32)
    assert not want.isnan().any() and (want[1, :T - T // 2] == 0).all()
    x = q.clone()
    x[:, 1::2, :, 3] = -math.inf
    got = shadowkv.kv8_attn(x, *caches, at, n, block=32)
    assert got[0, :, 1::2].isnan().all() and got[1, T - T // 2:, 1::2].isnan().all()
    assert (got[1, :T - T // 2] == 0).all() and not got[:, :, ::2].isnan().any()
    # (in 16 bits beside NaN, where the other call may have taken f16: 2^-11 of the values, and a bf16 rounding each)
    assert (got[:, :, ::2].float() - want[:, :, ::2].float()).abs().max() <= want.float().abs().max() * 2.0 ** -7 + \
        (caches[1].float().abs().amax() * caches[3].amax()) * 2.0 ** -10


@pytest.mark.parametrize("T,cap", [(1, 320), (1, 2500), (6, 320), (6, 2500), (50, 320), (50, 2500)])
@pytest.mark.parametrize("odd", [math.nan, math.inf])
def test_attn_seen_scales_that_are_not_finite(gpu, T, cap, odd):
    """A value block of a NaN or infinite scale makes the rows that see a key of it NaN also where the key's probability
    is too small for fp32 (zero times such a value), and no other rows."""
    _say(f"kv8_attn seen scales T={T} cap={cap} {odd}")
    g = torch.Generator().manual_seed(T)
    at, block = [300, 256], 16
    caches = _caches(2, 2, cap, block, g, gpu)
    far = [1, 17, (300 - T // 2) // block]  # blocks of tiny probabilities; the last is seen by some of the rows only
    k = torch.randn(2, 2, cap, D, generator=g)
    for j in far:
        k[:, :, j * block:(j + 1) * block] = -9.0
    v = torch.randn(2, 2, cap, D, generator=g)
    shadowkv.kv8_write(k.to(BF16).to(gpu), v.to(BF16).to(gpu), *caches, _ints([0, 0], gpu), block=block)
    q = torch.full((2, 8, T, D), 4.0).to(BF16).to(gpu)
    for window, sinks in ((None, 0), (40, 18)):
        for j in far:
            scales = caches[3].clone()
            scales[:, :, j] = odd
            got = shadowkv.kv8_attn(q, *caches[:3], scales, _ints(at, gpu), block=block, window=window, sinks=sinks).cpu()
            for b, L in enumerate(at):
                hit = _see(T, T, L, window, sinks)[:, torch.arange(L) // block == j].any(1)
                assert torch.equal(got[b].isnan().all(-1), hit.unsqueeze(1).expand(T, 8)), (b, j, window)
                assert torch.equal(got[b].isnan().any(-1), hit.unsqueeze(1).expand(T, 8)), (b, j, window)
