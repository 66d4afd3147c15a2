"""The edges of the 8-bit cache's attention: what lies behind a sequence's end, padding, scores and scales of every size,
and the many-row form's own paths (large workgroups without shares, more workgroups than the chip holds at once)."""
import math

import pytest
import torch

from shadowkv_amd import _lib
from shadowkv_amd.kernels import shadowkv

from .test_gpu_kv8 import BF16, D, E4M3, _caches, _check_write, _filled, _queries, _say, _see

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


def _check_sampled(q, caches, lengths, counts, block, window, sinks, rows):
    """kv8_attn's rows t of `rows` against 64 bits. Tolerance, from the many-row form with probabilities p_j (at most
    2^15, their largest at least 2^7) rounded to f16, p_j (1 + e_j) + z_j, |e_j| <= 2^-11, |z_j| <= 2^-25, over their own
    sum: (sum of w_j |v_j - out| 2^-11 + keys 2^-32 2 top) (1 + 2^-9), w the softmax, top the largest value; beside it
    twice a score's error (130 fp32 roundings of the sum of the products' magnitudes, 2^-22 for the exponential), the
    fp32 sums (2^-24 a key, numerator and denominator) and a few last roundings (2^-21), each of top; and the output's
    own rounding, 2^-8 of the value. (Two parts of bf16 are closer: 2^-15 of top would be left of the first term.)"""
    got, again = [shadowkv.kv8_attn(q, *caches, _ints(lengths, q.device), _ints(counts, q.device), block=block,
                                    window=window, sinks=sinks) for _ in range(2)]
    assert torch.equal(got.view(torch.int16), again.view(torch.int16))
    got = got.cpu().double()
    k8, v8, ks, vs = [c.cpu().double() for c in caches]
    B, Hq, T, _ = q.shape
    H, cap = k8.shape[1], k8.shape[2]
    G, rows = Hq // H, torch.tensor(rows)
    for b in range(B):
        L, n = min(lengths[b], cap), T if counts is None else counts[b]
        see = _see(n, T, L, window, sinks)[rows]
        none = ~see.any(1)
        assert (got[b, rows[none]] == 0).all()
        assert (got[b, n:] == 0).all()
        for h in range(H):
            kk = k8[b, h, :L] * ks[b, h].repeat_interleave(block)[:L, None]
            vv = v8[b, h, :L] * vs[b, h].repeat_interleave(block)[:L, None]
            clean, top = vv.nan_to_num(0.0), vv.nan_to_num(0.0).abs().max()
            for hq in range(h * G, (h + 1) * G):
                x = q[b, hq].cpu().double()[rows] / math.sqrt(D)
                w = torch.softmax((x @ kk.T).masked_fill(~see, -math.inf), -1).nan_to_num(0.0)
                want = w @ clean
                size = (x.abs() @ kk.abs().T).masked_fill(~see, 0.0).amax(1, keepdim=True)
                away = torch.stack([w[i] @ (clean - want[i]).abs() for i in range(len(rows))])
                tol = 2.0 ** -8 * want.abs() + 2.0 ** -11 * (1 + 2.0 ** -9) * away + top * (
                    L * 2.0 ** -31 + 2 * (130 * 2.0 ** -24 * size + 2.0 ** -22) + 2 * L * 2.0 ** -24 + 2.0 ** -21)
                nan = (see.double() @ vv.isnan().double()) > 0
                g = got[b, rows, hq]
                assert torch.equal(g.isnan(), nan), (b, hq)
                err = (g - want).abs().masked_fill(nan, 0.0)
                assert (err <= tol).all(), (b, hq, (err - tol).max(), err.max())


@pytest.mark.parametrize("T,cap,window,sinks", [(1000, 3000, None, 0), (1000, 3000, 2600, 40), (750, 760, None, 0),
                                                (750, 760, 200, 20)])
def test_attn_many_rows_direct(gpu, T, cap, window, sinks):
    """More workgroups than the chip holds at once, of 256 rows on long caches and of 128 on short ones, without shares
    of the keys: sequences of different lengths and counts, windows, NaN seen by some rows, scales that f16 does not
    hold together. Rows around the workgroups' and the waves' first and last."""
    _say(f"kv8_attn many rows direct T={T} cap={cap} window={window}")
    g = torch.Generator().manual_seed(T)
    B, H, G, block = 3, 8, 4, 32
    assert _lib.lib().skv_kv8_attn_workspace_bytes(B, H * G, H, T, cap, window or 0, sinks) == 0  # (no shares)
    q = _queries(B, H * G, T, g, gpu)
    caches = _filled(B, H, cap, block, g, gpu)
    lengths, counts = [cap, cap - 211, T + 5], [T, T - 130, T]
    rows = sorted({0, 1, 7, 8, 31, 32, 63, 64, 200, 333, 511, 512, T - 131, T - 130, T - 129, T - 64, T - 33, T - 2, T - 1})
    _check_sampled(q, caches, lengths, counts, block, window, sinks, rows)
    _check_sampled(q, caches, [T - 20, cap, 1], None, block, window, sinks, rows)
    v8 = caches[1].view(torch.uint8)
    for b, h, j, d in ((0, 0, cap - 40, 5), (0, 3, cap - T + 3, 127), (1, 7, lengths[1] - 300, 64), (2, 2, 9, 9)):
        v8[b, h, j, d] = 0x7f
    _check_sampled(q, caches, lengths, counts, block, window, sinks, rows)
    caches = _filled(B, H, cap, block, g, gpu)
    caches[3].mul_(torch.exp2(torch.randint(-9, 9, caches[3].shape, generator=g).float()).to(gpu))
    _check_sampled(q, caches, lengths, counts, block, window, sinks, rows)


@pytest.mark.parametrize("block", [16, 128])
def test_read_rows_from_the_host(gpu, block):
    """Rows of pinned host memory through kv8_read: the device cache's bits, from any first row, of other layouts too."""
    _say(f"kv8_read from the host block={block}")
    g = torch.Generator().manual_seed(block)
    k8, _, ks, _ = _caches(2, 3, 333, block, g, gpu)
    host = torch.empty(k8.shape, dtype=E4M3, pin_memory=True)
    side = torch.empty(2, 333, 3, D, dtype=E4M3, pin_memory=True).permute(0, 2, 1, 3)
    for c in (host, side):
        c.view(torch.uint8).copy_(k8.view(torch.uint8))
        for start, rows in ((0, 333), (17, 1), (100, 129), (332, 1)):
            want = shadowkv.kv8_read(k8, ks, start, rows, block=block)
            got = shadowkv.kv8_read(c, ks, start, rows, block=block)
            assert torch.equal(got.view(torch.int16), want.view(torch.int16))


def test_write_shared_memory(gpu):
    """Caches that overlap without beginning at the same place are refused; keys, values and scales that lie between
    one another in a buffer, and share nothing, are written as apart."""
    _say("kv8_write shared memory")
    g = torch.Generator().manual_seed(6)
    B, H, cap, block = 2, 2, 64, 32
    k, v = _queries(B, H, 40, g, gpu), _queries(B, H, 40, g, gpu)
    at = _ints([3, 20], gpu)
    buffer, scales = torch.zeros(B, H, 3 * cap, D, dtype=E4M3, device=gpu), torch.ones(B, H, 8, device=gpu)
    cut = lambda a: buffer[:, :, a:a + cap]  # noqa: E731
    for k8, v8, ks, vs in ((cut(0), cut(1), scales[..., :2], scales[..., 2:4]),
                           (cut(cap), cut(1), scales[..., :2], scales[..., 2:4]),
                           (cut(0), cut(cap), scales[..., :2], scales[..., 1:3]),
                           (cut(0), cut(cap), scales[..., 3:5], scales[..., 2:4]),
                           (buffer[:, :, :2 * cap:2], buffer[:, :, 2:2 * cap + 2:2], scales[..., :2], scales[..., 2:4])):
        with pytest.raises(ValueError, match="share memory"):
            shadowkv.kv8_write(k, v, k8, v8, ks, vs, at, block=block)
    assert buffer.view(torch.uint8).max() == 0 and (scales == 1).all()
    want = _caches(B, H, cap, block, g, gpu)
    start = [c.clone() for c in want]
    shadowkv.kv8_write(k, v, *want, at, block=block)
    records = torch.zeros(B, H, 2 * cap * D + 32, dtype=torch.uint8, device=gpu)  # a head's codes and scales together
    per = records.view(E4M3)[..., :2 * cap * D].unflatten(-1, (2, cap, D))
    tail = records.view(torch.float32)[..., 2 * cap * D // 4:]
    for k8, v8, ks, vs in ((cut(5), cut(5 + cap), scales[..., 1:3], scales[..., 4:6]),
                           (buffer[:, :, :2 * cap:2], buffer[:, :, 1:2 * cap + 1:2], scales[..., :2], scales[..., 2:4]),
                           (per[:, :, 0], per[:, :, 1], tail[..., :2], tail[..., 2:4])):
        for c, s in zip((k8, v8, ks, vs), start):
            c.copy_(s) if c.dtype != E4M3 else c.view(torch.uint8).copy_(s.view(torch.uint8))
        shadowkv.kv8_write(k, v, k8, v8, ks, vs, at, block=block)
        for c, w in zip((k8, v8, ks, vs), want):
            assert torch.equal(c.contiguous().view(torch.uint8), w.view(torch.uint8))


@pytest.mark.parametrize("block", [16, 64])
def test_write_beside_any_scale(gpu, block):
    """New rows in a block whose scale is no power of two (a cache that something else filled) and stays:
    the nearest code, ties to the even one. Odd scales, whose products with half steps are in bf16."""
    _say(f"kv8_write beside any scale block={block}")
    g = torch.Generator().manual_seed(block)
    H, cap = 120, 64
    scale = torch.ldexp((2.0 * torch.arange(H) + 3.0).view(1, H, 1), torch.randint(-20, 20, (1, H, 1), generator=g))
    caches = _caches(1, H, cap, block, g, gpu)
    for c in caches[2:]:
        c.copy_(scale.expand(-1, -1, c.shape[2]))
    ties = torch.arange(17, 32, 2).float() / 16  # half between two codes
    x = torch.where(torch.rand(1, H, 7, D, generator=g) < 0.7, ties[torch.randint(0, 8, (1, H, 7, D), generator=g)],
                    torch.randn(1, H, 7, D, generator=g).clamp(-3, 3))
    x = torch.ldexp(x * scale.unsqueeze(3), torch.randint(-8, 6, x.shape, generator=g)).to(BF16)
    _check_write(x.to(gpu), -x.to(gpu), caches, [5], None, block)


def test_scales_that_want_a_gradient(gpu):
    """The operators have no gradient, for scales neither, and say so."""
    _say("kv8 scales with gradients")
    g = torch.Generator().manual_seed(1)
    k8, v8, ks, vs = _caches(1, 2, 64, 32, g, gpu)
    x, at = _queries(1, 2, 3, g, gpu), _ints([9], gpu)
    ids = torch.zeros(1, 2, 1, dtype=torch.int64, device=gpu)
    for s, t in ((ks.clone().requires_grad_(), vs), (ks, vs.clone().requires_grad_())):
        for call in (lambda: shadowkv.kv8_write(x, x, k8, v8, s, t, at, block=32),
                     lambda: shadowkv.kv8_attn(x, k8, v8, s, t, at, block=32)):
            with pytest.raises(ValueError, match="gradient"):
                call()
    s = ks.clone().requires_grad_()
    for call in (lambda: shadowkv.kv8_read(k8, s, 0, 4, block=32),
                 lambda: shadowkv.kv8_read_chunks(k8, s, ids, 8, block=32)):
        with pytest.raises(ValueError, match="gradient"):
            call()
    with torch.no_grad():
        assert shadowkv.kv8_read(k8, s, 0, 4, block=32).shape == (1, 2, 4, D)
