"""Attention of packed rows over pages and over whole prompts (skv_paged_attn, skv_packed_attn) against 64 bits."""
import pytest
import torch

from shadowkv_amd.kernels import shadowkv
from shadowkv_amd.streams import capture_graph
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
INF, NAN = float("inf"), float("nan")


def _ints(v, gpu):
    return torch.tensor(v, dtype=torch.int32, device=gpu)


def _cu(counts, lead=0):
    out = [lead]
    for n in counts:
        out.append(out[-1] + n)
    return out


def _paged_case(gpu, lengths, counts, H, G, page, order="head", lead=0, pad=0, seed=0, width=0, spare=3, garbage=NAN):
    """q, pages and tables of sequences of `lengths` tokens; whatever no sequence holds is garbage."""
    gen = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lengths]
    P = sum(need) + spare
    ids = torch.randperm(P, generator=gen).to(torch.int32)
    table = torch.full((len(lengths), max(need + [1]) + width), -1, dtype=torch.int32)
    kp, vp = (torch.full((P, H, page, 128), garbage, dtype=BF16) for _ in range(2))
    at = 0
    chan = torch.exp(0.5 * torch.randn(1, H, 1, 128, generator=gen))
    for b, n in enumerate(lengths):
        mine = ids[at:at + need[b]]
        at += need[b]
        table[b, :need[b]] = mine
        x = torch.randn(need[b], H, page, 128, generator=gen) * chan
        y = torch.randn(need[b], H, page, 128, generator=gen) * 0.6 + 0.2
        if need[b] and n % page:
            x[-1, :, n % page:] = garbage
            y[-1, :, n % page:] = garbage
        kp[mine.long()], vp[mine.long()] = x.to(BF16), y.to(BF16)
    if order == "token":
        kp, vp = (x.transpose(1, 2).contiguous().to(gpu).transpose(1, 2) for x in (kp, vp))
    elif order == "pairs":
        x = torch.stack([kp, vp], 1).to(gpu)
        kp, vp = x[:, 0], x[:, 1]
    else:
        kp, vp = kp.to(gpu), vp.to(gpu)
    N = lead + sum(counts) + pad
    qkv = (1.2 * torch.randn(N, (G + 2) * H, 128, generator=gen)).to(BF16)
    cu = _cu(counts, lead)
    qkv[:lead], qkv[cu[-1]:] = garbage, garbage
    return dict(q=qkv.to(gpu)[:, :G * H], kp=kp, vp=vp, table=table.to(gpu), lengths=lengths, counts=counts, cu=cu,
                page=page)


def _expect_paged(c, window=None, scale=None):
    q = c["q"].cpu()
    outs = [torch.zeros(*q.shape, dtype=torch.float64) for _ in range(2)] + \
        [torch.zeros(*q.shape[:2], 1, dtype=torch.float64)]
    cap = c["table"].shape[1] * c["page"]
    for b, n in enumerate(c["counts"]):
        length = min(max(c["lengths"][b], 0), cap)
        if not n or not length:
            continue
        rows = slice(c["cu"][b], c["cu"][b] + n)
        k, there = ref.gathered(c["kp"], c["table"][b].cpu(), length, c["page"])
        v, _ = ref.gathered(c["vp"], c["table"][b].cpu(), length, c["page"])
        m = min(n, length)  # (those before the sequence see nothing)
        part = ref.attention(q[rows][n - m:], k, v, m, window, scale, there)
        for o, x in zip(outs, part):
            o[rows][n - m:] = x
    return outs


def _run_paged(c, gpu, max_new=None, window=None, scale=None, cu=True):
    return shadowkv.paged_attn(c["q"], c["kp"], c["vp"], c["table"], _ints(c["lengths"], gpu),
                               _ints(c["cu"], gpu) if cu else None, max_new=max_new, window=window, scale=scale)


def _bits(c, max_new):
    """Significant bits of a probability in every form that the call may take."""
    G = c["q"].shape[1] // c["kp"].shape[1]
    return 16 if max_new is not None and max_new * G <= 32 else 8


@pytest.mark.parametrize("page,order", [(16, "head"), (64, "token"), (256, "pairs"), (32, "head"), (128, "token")])
@pytest.mark.parametrize("H,G", [(1, 1), (2, 4), (1, 7), (1, 16), (2, 2)])
def test_tokens(gpu, page, order, H, G):
    """One token of each sequence, of lengths around the groups', chunks' and pages' ends."""
    lengths = [1, 2, 15, 16, 17, 31, 33, 64, 65, 255, 257, 700, 0]
    c = _paged_case(gpu, lengths, [1] * len(lengths), H, G, page, order, seed=page + H)
    got = _run_paged(c, gpu, cu=False)
    ref.check(got, *_expect_paged(c), bits=16)
    assert torch.equal(got, _run_paged(c, gpu, max_new=1)), "the same rows, with cu"


@pytest.mark.parametrize("H,G", [(2, 4), (1, 16), (1, 32)])
def test_tokens_of_long_sequences(gpu, H, G):
    """Chunks and their join; tables that end far behind."""
    c = _paged_case(gpu, [5000, 1, 2047, 3001], [1] * 4, H, G, 64, seed=G, width=300)
    ref.check(_run_paged(c, gpu, cu=False), *_expect_paged(c), bits=16)


@pytest.mark.parametrize("window", [1, 16, 63, 500, 2 ** 31 - 1])
def test_window(gpu, window):
    c = _paged_case(gpu, [1, 40, 700, 1500], [1, 1, 1, 1], 1, 4, 32, seed=window % 97)
    ref.check(_run_paged(c, gpu, cu=False, window=window), *_expect_paged(c, window), bits=16)
    c = _paged_case(gpu, [5, 40, 700, 1500], [5, 3, 4, 1], 1, 4, 32, seed=window % 97, lead=1, pad=2)
    ref.check(_run_paged(c, gpu, max_new=5, window=window), *_expect_paged(c, window), bits=16)
    c = _paged_case(gpu, [50, 140, 700, 900], [50, 33, 70, 1], 1, 4, 32, seed=window % 97, pad=1)
    ref.check(_run_paged(c, gpu, window=window), *_expect_paged(c, window), bits=8)


@pytest.mark.parametrize("counts,lengths,max_new", [
    ([1], [1], 1), ([2, 5, 0, 1], [2, 90, 33, 64], 5), ([8, 8], [8, 1200], 8), ([3, 8, 1, 1], [3, 8, 0, 5000], 8),
    ([4, 0, 0, 2], [100, 0, 7, 2], 4)])
@pytest.mark.parametrize("H,G", [(1, 4), (2, 2), (1, 3)])
def test_drafts(gpu, counts, lengths, max_new, H, G):
    """Several new tokens, up to 32 rows; rows in front of the first sequence and behind the last; sequences of no new
    tokens, of no tokens, and of fewer than are new."""
    c = _paged_case(gpu, lengths, counts, H, G, 16, "token", lead=3, pad=5, seed=sum(lengths))
    got = _run_paged(c, gpu, max_new=max_new)
    ref.check(got, *_expect_paged(c), bits=_bits(c, max_new))
    assert not got[:3].any() and not got[-5:].any()


@pytest.mark.parametrize("counts,lengths", [
    ([33], [33]), ([128], [128]), ([129, 1], [129, 300]), ([64, 200, 3], [500, 200, 3]), ([1, 1, 90, 1], [900, 1, 150, 64]),
    ([97, 0, 65], [97, 4, 129]), ([40, 50], [30, 700])])
@pytest.mark.parametrize("H,G,page", [(1, 4, 16), (2, 1, 64), (1, 7, 128), (1, 48, 32)])
def test_pieces(gpu, counts, lengths, H, G, page):
    """Pieces of prompts beside single tokens: both forms in one call."""
    c = _paged_case(gpu, lengths, counts, H, G, page, lead=2, pad=3, seed=sum(lengths) + G)
    got = _run_paged(c, gpu)
    ref.check(got, *_expect_paged(c), bits=8)
    assert not got[:2].any() and not got[-3:].any()


def test_piece_of_a_long_sequence_is_shared_out(gpu):
    """Few rows of long sequences, in shares of the keys that are joined."""
    c = _paged_case(gpu, [3000, 70, 1900], [40, 3, 1], 1, 4, 64, seed=5, pad=1)
    ref.check(_run_paged(c, gpu), *_expect_paged(c), bits=8)
    c = _paged_case(gpu, [2500], [37], 2, 2, 16, "token", seed=6)
    ref.check(_run_paged(c, gpu), *_expect_paged(c), bits=8)


@pytest.mark.parametrize("counts,lengths,page", [([600], [600], 64), ([515, 1, 37], [700, 300, 4200], 16),
                                                 ([130, 400], [131, 401], 256)])
@pytest.mark.parametrize("window", [None, 150])
def test_pieces_in_wide_tables(gpu, counts, lengths, page, window):
    """Tables of 4096 tokens and more, rows enough: 256 rows a workgroup."""
    c = _paged_case(gpu, lengths, counts, 4, 8, page, "token", lead=1, pad=2, seed=sum(counts), width=4096 // page)
    ref.check(_run_paged(c, gpu, window=window), *_expect_paged(c, window), bits=8)


def test_values_and_pages_in_wide_tables(gpu):
    """NaN and infinities, pages that do not exist, scores of every size: with 256 rows a workgroup."""
    c = _paged_case(gpu, [600, 90], [540, 1], 2, 16, 64, seed=5, width=64)
    page = lambda j: (int(c["table"][0, j // 64]), 1, j % 64)  # noqa: E731
    for j, d, x in ((599, 3, NAN), (598, 5, INF), (300, 5, -INF), (61, 6, -INF), (130, 127, NAN)):
        c["vp"][page(j)][d] = x
    ref.check(_run_paged(c, gpu), *_expect_paged(c), bits=8)
    c = _paged_case(gpu, [600, 90], [540, 1], 2, 16, 64, seed=6, width=64)
    c["table"][0, 3], c["table"][0, 9] = -1, 10 ** 6
    ref.check(_run_paged(c, gpu), *_expect_paged(c), bits=8)
    c = _paged_case(gpu, [600, 90], [540, 1], 2, 16, 64, seed=7, width=64)
    c["q"][:], c["kp"][:] = 0, 0
    c["q"][:, :, 0], c["kp"][..., 0] = 2.0 ** 20 * 128 ** 0.5, 2.0 ** 20
    out, mean, _ = _expect_paged(dict(c, q=torch.zeros_like(c["q"])))
    ref.check(_run_paged(c, gpu), out, mean, torch.zeros(*out.shape[:2], 1, dtype=torch.float64), bits=8)


def test_a_few_rows_of_a_long_sequence_in_wide_tables(gpu):
    """Shares of the keys and their join with 256 rows a workgroup, with more than 16 shares and with fewer."""
    for counts, lengths in (([520], [4300]), ([300, 300], [3000, 2500])):
        c = _paged_case(gpu, lengths, counts, 1, 32, 64, seed=lengths[0], width=10)
        ref.check(_run_paged(c, gpu), *_expect_paged(c), bits=8)


@pytest.mark.parametrize("B", [64, 65, 150])
def test_many_sequences(gpu, B):
    """More sequences than a wave has lanes: single tokens, drafts, pieces beside them, chunks and shares among them."""
    lengths = [1 + (37 * b) % 90 for b in range(B)]
    lengths[3], lengths[B - 1], lengths[63] = 1500, 1900, 700
    c = _paged_case(gpu, lengths, [1] * B, 1, 4, 16, seed=B, width=40)
    ref.check(_run_paged(c, gpu, cu=False), *_expect_paged(c), bits=16)
    counts = [min(n, b % 4) for b, n in enumerate(lengths)]
    c = _paged_case(gpu, lengths, counts, 1, 4, 16, seed=B, lead=2, pad=3)
    ref.check(_run_paged(c, gpu, max_new=3), *_expect_paged(c), bits=16)
    counts[3], counts[B - 1], counts[63], counts[40] = 45, 70, 60, lengths[40]
    c = _paged_case(gpu, lengths, counts, 1, 4, 16, seed=B, lead=2, pad=3)
    ref.check(_run_paged(c, gpu), *_expect_paged(c), bits=8)


def test_many_shares(gpu):
    """More than 16 shares of a row tile, under a window too; of rows under a window."""
    c = _paged_case(gpu, [6000, 200], [40, 1], 1, 4, 64, seed=9, pad=1)
    ref.check(_run_paged(c, gpu), *_expect_paged(c), bits=8)
    ref.check(_run_paged(c, gpu, window=5000), *_expect_paged(c, 5000), bits=8)
    c = _paged_case(gpu, [4000], [130], 1, 4, 64, seed=10)
    ref.check(_run_paged(c, gpu, window=1500), *_expect_paged(c, 1500), bits=8)


def test_more_new_tokens_than_the_host_said(gpu):
    """A sequence with more than max_new gives zeros, the others what they give."""
    c = _paged_case(gpu, [50, 40, 90], [2, 9, 1], 1, 4, 16, seed=8)
    whole = _expect_paged(dict(c, counts=[2, 9, 1]))
    for o in whole:
        o[2:11] = 0
    ref.check(_run_paged(c, gpu, max_new=4), *whole, bits=16)
    c = _paged_case(gpu, [50, 140, 90], [2, 99, 40], 1, 4, 16, seed=9)
    whole = _expect_paged(c)
    for o in whole:
        o[2:101] = 0
    ref.check(_run_paged(c, gpu, max_new=40), *whole, bits=8)


@pytest.mark.parametrize("counts,max_new", [([1, 1, 1, 1], 1), ([2, 1, 4, 3], 4), ([60, 2, 50, 1], None)])
def test_pages_that_do_not_exist(gpu, counts, max_new):
    """Keys of pages outside the pool are not seen: holes, the first page, all of a sequence, far-off numbers."""
    c = _paged_case(gpu, [100, 300, 64, 700], counts, 1, 4, 16, seed=3)
    t = c["table"]
    P = c["kp"].shape[0]
    t[0, 0], t[0, 6], t[1, 3], t[1, 18] = -1, P, 2 ** 31 - 1, -2 ** 31
    t[2, :] = -1
    t[3, 5:30] = P + 1
    got = _run_paged(c, gpu, max_new=max_new)
    ref.check(got, *_expect_paged(c), bits=_bits(c, max_new))
    assert not got[c["cu"][2]:c["cu"][3]].any()


@pytest.mark.parametrize("n,max_new,G", [(5, 5, 4), (3, 3, 8), (70, None, 2), (150, None, 1)])
def test_values_that_are_no_numbers(gpu, n, max_new, G):
    """NaN and infinities of both signs reach the queries that see their keys and no others, with and without a window,
    also where the keys before make their probabilities small."""
    c = _paged_case(gpu, [n + 61, 200], [n, 1], 1, G, 64, seed=n)
    L = n + 61
    page = lambda j: (int(c["table"][0, j // 64]), 0, j % 64)  # noqa: E731
    for j, d, x in ((L - 1, 3, NAN), (L - 2, 5, INF), (L - 2, 6, -INF), (L - n + 1, 7, INF), (L - 1, 7, -INF),
                    (L - n, 100, -INF), (L - 2, 127, NAN)):
        c["vp"][page(j)][d] = x
    got = _run_paged(c, gpu, max_new=max_new)
    ref.check(got, *_expect_paged(c), bits=_bits(c, max_new))
    c["vp"][page(40)][64] = NAN
    for window in (30, L - 41):  # (the second: the last query no longer sees key 40)
        ref.check(_run_paged(c, gpu, max_new=max_new, window=window), *_expect_paged(c, window), bits=_bits(c, max_new))


@pytest.mark.parametrize("n,max_new", [(4, 4), (80, None)])
def test_keys_that_are_no_numbers(gpu, n, max_new):
    """A NaN key makes those that see it NaN; scores of -inf take no part, of -inf alone are NaN."""
    c = _paged_case(gpu, [n + 30, n], [n, n], 1, 4, 32, seed=n)
    c["q"][:, :, 0] = 1.0
    c["kp"][int(c["table"][0, (n + 28) // 32]), 0, (n + 28) % 32, 1] = NAN
    first = int(c["table"][1, 0])
    c["kp"][first, 0, 0, 0] = -INF
    c["kp"][first, 0, 1, 0] = -INF
    got = _run_paged(c, gpu, max_new=max_new)
    ref.check(got, *_expect_paged(c), bits=_bits(c, max_new))
    assert got[n:n + 2].isnan().all() and got[n - 2:n].isnan().all()
    assert got[:n - 2].isfinite().all() and got[n + 2:].isfinite().all()


@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-30, 40.0])
@pytest.mark.parametrize("counts,max_new", [([1, 3], 3), ([70, 40], None)])
def test_scales(gpu, scale, counts, max_new):
    c = _paged_case(gpu, [300, 77], counts, 1, 4, 16, seed=2)
    ref.check(_run_paged(c, gpu, max_new=max_new, scale=scale), *_expect_paged(c, scale=scale), bits=_bits(c, max_new))


@pytest.mark.parametrize("counts,max_new", [([2, 3], 3), ([70, 40], None)])
def test_scores_of_every_size(gpu, counts, max_new):
    """Equal scores of up to 2^40 give the mean of the values."""
    for size in (2.0 ** 8, 2.0 ** 26, 2.0 ** 40):
        c = _paged_case(gpu, [300, 77], counts, 1, 4, 16, seed=4)
        c["q"][:], c["kp"][:] = 0, 0
        c["q"][:, :, 0], c["kp"][..., 0] = size ** 0.5 * 128 ** 0.5, size ** 0.5
        out, mean, _ = _expect_paged(dict(c, q=torch.zeros_like(c["q"])))
        ref.check(_run_paged(c, gpu, max_new=max_new), out, mean, torch.zeros(*out.shape[:2], 1, dtype=torch.float64),
                  bits=_bits(c, max_new))


def test_bad_lengths_and_places_stay_in_bounds(gpu):
    """Lengths outside the table are clamped to it, places outside the rows to them."""
    for counts, max_new in (([1, 2, 1, 1], 2), ([50, 2, 40, 1], None)):
        c = _paged_case(gpu, [200, 200, 200, 200], counts, 1, 4, 16, seed=7)
        c["lengths"] = [2 ** 31 - 1, -5, 208, -2 ** 31]
        for x in ("kp", "vp"):
            c[x][c[x].isnan()] = 0.5
        ref.check(_run_paged(c, gpu, max_new=max_new), *_expect_paged(c), bits=_bits(c, max_new))
        N = c["q"].shape[0]
        for cu in ([-7, 1, 2, 3, N + 100], [2 ** 31 - 1] * 5, [N, 3, 2, 1, 0], [-2 ** 31, 2 ** 31 - 1, 0, 1, 2]):
            _run_paged(dict(c, cu=cu), gpu, max_new=max_new)
        torch.cuda.synchronize()


def test_shared_pages(gpu):
    """Two sequences with the same first pages, and one table row in one page twice."""
    c = _paged_case(gpu, [150, 170], [20, 1], 1, 4, 16, seed=12)
    c["table"][1, :5] = c["table"][0, :5]
    c["table"][1, 7] = c["table"][1, 6]
    ref.check(_run_paged(c, gpu), *_expect_paged(c), bits=8)


def test_pool_of_more_than_2_to_the_31_elements(gpu):
    H, page = 8, 256
    P = 2 ** 31 // (H * page * 128) + 9
    c = _paged_case(gpu, [500, 900], [1, 1], H, 2, page, seed=1)
    kp, vp = (torch.empty(P, H, page, 128, dtype=BF16, device=gpu) for _ in range(2))
    shift = P - c["kp"].shape[0]
    kp[shift:], vp[shift:] = c["kp"], c["vp"]
    far = dict(c, kp=kp, vp=vp, table=torch.where(c["table"] < 0, -1, c["table"] + shift))
    assert torch.equal(_run_paged(far, gpu, cu=False), _run_paged(c, gpu, cu=False))
    c = _paged_case(gpu, [500, 900], [64, 50], H, 2, page, seed=1)
    kp[shift:], vp[shift:] = c["kp"], c["vp"]
    far = dict(c, kp=kp, vp=vp, table=torch.where(c["table"] < 0, -1, c["table"] + shift))
    assert torch.equal(_run_paged(far, gpu), _run_paged(c, gpu))


@pytest.mark.parametrize("n", [37, 130])
def test_shares_of_plans_past_2_to_the_24_tiles(gpu, n):
    """Row tiles of sequences of some 2^24 tokens, each a page of its own over and over: the plan's sums are rounded, and the
    join finds the shares that the kernel made. (Equal values: sums of multiples of two below 2^24, exact.)"""
    page, width, B = 256, 2 ** 16, 7
    table = torch.arange(B, dtype=torch.int32, device=gpu).unsqueeze(1).expand(B, width).contiguous()
    value = 1 + torch.arange(B, device=gpu) / 8
    kp = torch.randn(B, 1, page, 128, generator=torch.Generator().manual_seed(0)).to(BF16).to(gpu)
    vp = value.to(BF16).view(B, 1, 1, 1).expand(B, 1, page, 128).contiguous()
    q = torch.zeros(B * n, 32, 128, dtype=BF16, device=gpu)
    lengths = [2 ** 24 - 12345 * b * b for b in range(B)]
    out = shadowkv.paged_attn(q, kp, vp, table, _ints(lengths, gpu), _ints(_cu([n] * B), gpu), max_new=n)
    assert torch.equal(out.float(), value.repeat_interleave(n).view(-1, 1, 1).expand(-1, 32, 128))


def _far_apart(c, b, first, size):
    """Scores of sequence b's first keys some 600 (log2) below those behind, at values of that size."""
    c["q"][:, :, 0] = 16.0
    for j in range(c["lengths"][b]):
        at = int(c["table"][b, j // c["page"]]), slice(None), j % c["page"]
        c["kp"][at][:, 0] = 0.0 if j < first else 300.0
        if j < first:
            c["vp"][at] = torch.where(c["vp"][at] > 0, size, -size).to(BF16)


@pytest.mark.parametrize("lengths,counts,max_new", [([500, 90], [1, 1], 1), ([300, 90], [5, 2], 5), ([4000, 90], [1, 1], 1),
                                                    ([4000, 90], [5, 2], 5), ([400, 90], [70, 2], None),
                                                    ([4200, 90], [70, 2], None), ([5000], [37], None)])
def test_large_values_of_small_probabilities(gpu, lengths, counts, max_new):
    """Values of 10^36 whose probabilities underflow add nothing, in any form, share or join (sums of 250: below 3e38)."""
    for first in (1, 130, 250):
        c = _paged_case(gpu, lengths, counts, 1, 4, 64, seed=first)
        _far_apart(c, 0, first, 1e36)
        ref.check(_run_paged(c, gpu, max_new=max_new), *_expect_paged(c), bits=_bits(c, max_new))


@pytest.mark.parametrize("n,max_new,G", [(1, 1, 4), (6, 6, 4), (80, None, 4), (600, None, 16)])
def test_a_value_near_the_largest(gpu, n, max_new, G):
    """Of a score 7 (log2) above the others': its share of the sum, finite as the sum is."""
    c = _paged_case(gpu, [n + 200, 90], [n, 1], 2, G, 64, seed=n, width=64)
    c["q"][:], c["kp"][:] = 0, 0
    c["q"][:, :, 0] = 1.0
    at = int(c["table"][0, 2]), slice(None), 5
    c["kp"][at][:, 0] = 55.0
    c["vp"][at][:, :60] = 2.5e38
    ref.check(_run_paged(c, gpu, max_new=max_new), *_expect_paged(c), bits=_bits(c, max_new))


@pytest.mark.parametrize("counts,max_new", [([2, 3], 3), ([70, 40], None)])
def test_scale_of_zero_at_large_products(gpu, counts, max_new):
    """The mean of the values, whatever the products of queries and keys are."""
    c = _paged_case(gpu, [300, 77], counts, 1, 4, 16, seed=4)
    c["q"][:, :, 0], c["kp"][..., 0] = 1e19, c["kp"][..., 0].sign() * 1e19
    for scale in (0.0, -0.0, 1e-45):
        ref.check(_run_paged(c, gpu, max_new=max_new, scale=scale), *_expect_paged(c, scale=0.0), bits=_bits(c, max_new))


def test_sequences_of_2_to_the_31_groups_together(gpu):
    """64 sequences of as many tokens as a table can hold, all of them one page, over and over: the mean of equal values.
    (Sums of ones, below 2^24 in a wave: exact.)"""
    page, width = 256, shadowkv.PAGED_MAX_TOKENS // 256
    table = torch.zeros(1, width, dtype=torch.int32, device=gpu).expand(64, width)
    kp = torch.randn(1, 1, page, 128, generator=torch.Generator().manual_seed(0)).to(BF16).to(gpu)
    vp = torch.ones_like(kp)
    q = torch.zeros(64, 1, 128, dtype=BF16, device=gpu)
    out = shadowkv.paged_attn(q, kp, vp, table, _ints([shadowkv.PAGED_MAX_TOKENS] * 64, gpu))
    assert bool((out == 1).all())


def test_the_same_bits_each_time_and_on_another_stream(gpu):
    for counts, max_new in (([1, 1, 3], 3), ([90, 1, 200], None)):
        c = _paged_case(gpu, [2000, 5000, 900], counts, 2, 4, 64, seed=3)
        a = _run_paged(c, gpu, max_new=max_new)
        side = torch.cuda.Stream(gpu)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            b = _run_paged(c, gpu, max_new=max_new)
        other = _run_paged(c, gpu, max_new=max_new)  # (at once with it)
        torch.cuda.synchronize()
        assert torch.equal(a, b) and torch.equal(a, other)


@pytest.mark.parametrize("most,max_new", [(2, 2), (64, None)])
def test_captured_calls_follow_lengths_and_counts(gpu, most, max_new):
    """Two graphs of one shape, replayed in turn while lengths, places and tables change beneath them."""
    lengths, counts = [700, 40, 1300], [most, 1, most]
    c = _paged_case(gpu, lengths, counts, 1, 4, 64, seed=5, pad=2)
    cu, ln = _ints(c["cu"], gpu), _ints(lengths, gpu)
    q = c["q"].contiguous()

    def call():
        return shadowkv.paged_attn(q, c["kp"], c["vp"], c["table"], ln, cu, max_new=max_new)

    call()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with capture_graph(g, gpu):
            outs.append(call())
        graphs.append(g)
    for i, (ln_now, counts_now) in enumerate(((lengths, counts), ([650, 33, 1299], [1, most, 1]), ([64, 0, 9], [0, 1, most]),
                                              (lengths, counts))):
        ln.copy_(_ints(ln_now, gpu))
        cu.copy_(_ints(_cu(counts_now), gpu))
        graphs[i % 2].replay()
        graphs[1 - i % 2].replay()
        eager = call()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], eager) and torch.equal(outs[1], eager)
        assert not eager[sum(counts_now):].any()


# ---- whole prompts --------------------------------------------------------------------------------


def _packed_case(gpu, counts, H, G, lead=0, pad=0, seed=0):
    gen = torch.Generator().manual_seed(seed)
    N = lead + sum(counts) + pad
    qkv = 1.2 * torch.randn(N, (G + 2) * H, 128, generator=gen)
    qkv[:, G * H:(G + 1) * H] *= torch.exp(0.5 * torch.randn(1, H, 128, generator=gen))
    cu = _cu(counts, lead)
    qkv[:lead], qkv[cu[-1]:] = NAN, NAN
    qkv = qkv.to(BF16).to(gpu)
    return qkv.split([G * H, H, H], 1) + (cu, counts)


def _expect_packed(case, window=None, scale=None):
    q, k, v, cu, counts = case
    outs = [torch.zeros(*q.shape, dtype=torch.float64) for _ in range(2)] + \
        [torch.zeros(*q.shape[:2], 1, dtype=torch.float64)]
    for b, n in enumerate(counts):
        rows = slice(cu[b], cu[b] + n)
        if n:
            kk, vv = (x[rows].cpu().double().transpose(0, 1) for x in (k, v))
            for o, x in zip(outs, ref.attention(q[rows], kk, vv, n, window, scale)):
                o[rows] = x
    return outs


def _run_packed(case, gpu, **kw):
    q, k, v, cu, _ = case
    return shadowkv.packed_attn(q, k, v, _ints(cu, gpu), **kw)


@pytest.mark.parametrize("counts", [[1], [2, 1, 63], [64, 65], [128, 0, 129, 1], [300, 31, 1, 200], [33] * 9])
@pytest.mark.parametrize("H,G", [(1, 1), (2, 4), (1, 7), (1, 16), (1, 130)])
def test_prompts(gpu, counts, H, G):
    if G == 130:
        counts = [min(n, 40) for n in counts]
    case = _packed_case(gpu, counts, H, G, lead=2, pad=3, seed=sum(counts) + G)
    got = _run_packed(case, gpu)
    ref.check(got, *_expect_packed(case), bits=8)
    assert not got[:2].any() and not got[-3:].any()


@pytest.mark.parametrize("window", [1, 17, 64, 200, 2 ** 31 - 1])
def test_prompts_window(gpu, window):
    case = _packed_case(gpu, [400, 3, 130], 1, 4, pad=1, seed=window % 89)
    ref.check(_run_packed(case, gpu, window=window), *_expect_packed(case, window), bits=8)


@pytest.mark.parametrize("counts,H,G", [([1100, 4], 1, 1), ([2000], 2, 1), ([900, 1300, 700], 1, 2)])
def test_prompt_in_shares(gpu, counts, H, G):
    """Prompts of too few row tiles to fill the chip: the later ones' keys in shares, each its own number."""
    case = _packed_case(gpu, counts, H, G, seed=3)
    ref.check(_run_packed(case, gpu), *_expect_packed(case), bits=8)


def test_many_prompts(gpu):
    counts = [1 + (29 * b) % 60 for b in range(140)]
    counts[70], counts[139], counts[2] = 900, 850, 0
    case = _packed_case(gpu, counts, 1, 3, lead=1, pad=1, seed=4)
    ref.check(_run_packed(case, gpu), *_expect_packed(case), bits=8)


@pytest.mark.parametrize("counts,H,G", [([1100], 2, 64), ([1030, 1041], 8, 8), ([2100, 300], 1, 56)])
def test_long_prompts(gpu, counts, H, G):
    """Rows and tokens enough for 256 rows a workgroup."""
    case = _packed_case(gpu, counts, H, G, lead=1, pad=2, seed=counts[0])
    got = _run_packed(case, gpu)
    assert not got[:1].any() and not got[-2:].any()
    ref.check(got, *_expect_packed(case), bits=8)
    if G == 64:
        ref.check(_run_packed(case, gpu, window=333), *_expect_packed(case, 333), bits=8)


def test_prompt_values_that_are_no_numbers(gpu):
    case = _packed_case(gpu, [200, 90], 1, 4, seed=6)
    q, k, v, cu, counts = case
    for r, d, x in ((150, 1, NAN), (150, 2, INF), (199, 2, -INF), (0, 3, -INF), (289, 4, NAN), (230, 5, INF)):
        v[r, 0, d] = x
    ref.check(_run_packed(case, gpu), *_expect_packed(case), bits=8)
    ref.check(_run_packed(case, gpu, window=40), *_expect_packed(case, 40), bits=8)


def test_prompts_of_other_strides(gpu):
    """Rows that cannot be read 16 bytes at a time, heads outside rows, one kv head expanded."""
    gen = torch.Generator().manual_seed(1)
    q = torch.randn(4, 70, 128, generator=gen).to(BF16).to(gpu).transpose(0, 1)
    k = torch.randn(70, 2, 129, generator=gen).to(BF16).to(gpu)[..., 1:]
    v = torch.randn(70, 1, 128, generator=gen).to(BF16).to(gpu).expand(70, 2, 128)
    case = q, k, v, [0, 50, 70], [50, 20]
    ref.check(_run_packed(case, gpu), *_expect_packed(case), bits=8)


def test_prompts_equal_their_pages(gpu):
    """Prompts written into pages and read from there give what they give from their rows, to the bit."""
    counts = [200, 77, 1, 130]
    q, k, v, cu, _ = _packed_case(gpu, counts, 2, 4, seed=9)
    page, B = 16, len(counts)
    table = torch.full((B, 16), -1, dtype=torch.int32, device=gpu)
    free = torch.randperm(40, generator=torch.Generator().manual_seed(0)).to(torch.int32).to(gpu)
    held, count, lengths = _ints([0] * B, gpu), _ints([40], gpu), _ints([0] * B, gpu)
    kp, vp = (torch.full((40, 2, page, 128), NAN, dtype=BF16, device=gpu) for _ in range(2))
    places, totals, slots = shadowkv.paged_reserve(lengths, _ints(counts, gpu), table, held, free, count,
                                                   rows=sum(counts), page=page)
    shadowkv.paged_write(k, v, kp, vp, slots)
    got = shadowkv.paged_attn(q[:201], kp, vp, table[:1], totals[:1], _ints([0, 200], gpu))
    assert torch.equal(got[:200], shadowkv.packed_attn(q[:200], k[:200], v[:200], _ints([0, 200], gpu)))
    assert places.tolist() == cu
    want = _expect_packed((q, k, v, cu, counts))
    ref.check(shadowkv.paged_attn(q, kp, vp, table, totals, places), *want, bits=8)
    ref.check(shadowkv.packed_attn(q, k, v, places), *want, bits=8)


def test_captured_prompts(gpu):
    q, k, v, cu, counts = _packed_case(gpu, [90, 130, 20], 1, 4, seed=2)
    places = _ints(cu, gpu)
    shadowkv.packed_attn(q, k, v, places)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with capture_graph(g, gpu):
        out = shadowkv.packed_attn(q, k, v, places)
    for now in (cu, [0, 1, 2, 3], [5, 5, 200, 240], cu):
        places.copy_(_ints(now, gpu))
        g.replay()
        eager = shadowkv.packed_attn(q, k, v, places)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


def test_no_rows(gpu):
    c = _paged_case(gpu, [10], [1], 1, 4, 16)
    assert shadowkv.paged_attn(c["q"][:0], c["kp"], c["vp"], c["table"], _ints([10], gpu), _ints([0, 0], gpu)).shape == \
        (0, 4, 128)
    x = c["q"][:0]
    assert shadowkv.packed_attn(x, x, x, _ints([0, 0], gpu)).shape == (0, 4, 128)
