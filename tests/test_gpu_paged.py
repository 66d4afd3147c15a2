"""Page tables, slots and the write of a paged KV cache (skv_paged_reserve, skv_paged_release, skv_paged_write)."""
import random

import pytest
import torch

from shadowkv_amd.kernels import shadowkv
from shadowkv_amd.streams import capture_graph
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _ints(v, gpu):
    return torch.tensor(v, dtype=torch.int32, device=gpu)


class State:
    """Lists beside the device's copy of them."""

    def __init__(self, lengths, width, page, spare, rng, gpu, extra=0):
        need = [-(-max(n, 0) // page) for n in lengths]
        ids = list(range(sum(need) + spare))
        rng.shuffle(ids)
        self.page, self.lengths, self.held = page, list(lengths), need
        self.table, at = [], 0
        for n in need:
            self.table.append(ids[at:at + n] + [-1] * (width - n))
            at += n
        self.free, self.total = ids[at:], len(ids)
        whole = torch.full((len(lengths), width + extra), -7, dtype=torch.int32, device=gpu)  # a view of a wider one
        whole[:, :width] = _ints(self.table, gpu).view(len(lengths), width)
        self.whole, self.t_table = whole, whole[:, :width]
        self.t_held, self.t_lengths = _ints(self.held, gpu), _ints(self.lengths, gpu)
        self.t_free = _ints(self.free + [-5] * (max(1, self.total) - len(self.free)), gpu)
        self.t_count = _ints([len(self.free)], gpu)

    def args(self):
        return self.t_table, self.t_held, self.t_free, self.t_count

    def check(self):
        assert self.t_table.tolist() == self.table
        assert self.t_held.tolist() == self.held
        assert self.t_lengths.tolist() == self.lengths
        assert self.t_count.item() == len(self.free)
        assert self.t_free[:len(self.free)].tolist() == self.free
        assert bool((self.whole[:, self.t_table.shape[1]:] == -7).all())


def _step(st, counts, rows, gpu):
    cu, totals, slots = shadowkv.paged_reserve(st.t_lengths, _ints(counts, gpu), *st.args(), rows=rows, page=st.page)
    want = ref.reserve(st.lengths, counts, st.table, st.held, st.free, rows, st.page)
    assert (cu.tolist(), totals.tolist(), slots.tolist()) == want
    st.check()
    return totals.tolist()


def _back(st, keep, gpu):
    shadowkv.paged_release(st.t_lengths, st.t_lengths if keep is None else _ints(keep, gpu), *st.args(), page=st.page)
    ref.release(st.lengths, list(st.lengths) if keep is None else keep, st.table, st.held, st.free, st.page)
    st.check()


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("B,most,rows_each,pad", [(1, 1, 1, 0), (3, 100, 40, 5), (64, 3000, 1, 0), (65, 500, 90, 17),
                                                  (1500, 200, 3, 1), (40, 700, 301, 100)])
def test_steps_taken_given_back_and_kept(gpu, page, B, most, rows_each, pad):
    """A step is reserved, reserved again, taken back to the bit, reserved and kept, cut to shorter lengths."""
    rng = random.Random(B * page)
    lengths = [rng.randrange(most) for _ in range(B)]
    width = -(-(most + 2 * rows_each) // page) + 1
    st = State(lengths, width, page, B * (rows_each // page + 2), rng, gpu, extra=3)
    counts = [rng.choice([0, 1, rows_each, -2]) for _ in range(B)]
    rows = sum(max(c, 0) for c in counts) + pad
    before = (st.t_table.tolist(), st.t_held.tolist(), st.t_free.tolist(), st.t_count.item())
    _step(st, counts, rows, gpu)
    _step(st, counts, rows, gpu)
    _back(st, None, gpu)
    assert before == (st.t_table.tolist(), st.t_held.tolist(), st.t_free.tolist(), st.t_count.item())
    totals = _step(st, counts, rows, gpu)
    st.lengths = [max(n, t) for n, t in zip(st.lengths, totals)]
    st.t_lengths.copy_(_ints(st.lengths, gpu))
    _back(st, [rng.choice([-1, 0, n // 2, n, n + 5]) for n in st.lengths], gpu)
    _step(st, counts, rows, gpu)
    _back(st, [0] * B, gpu)
    assert len(st.free) == st.total


@pytest.mark.parametrize("rows", [64, 5000])
def test_what_cannot_be_served_is_left(gpu, rows):
    """Too few free pages (the first that lacks one and all that lack any behind it), tables too narrow, negative lengths,
    more tokens than rows."""
    rng = random.Random(rows)
    for spare, lengths, counts in (
            (3, [10, 16, 31, 32, 5], [6, 1, 2, 40, 1]), (0, [16, 15, 0], [1, 1, 1]), (1, [16, 16, 16], [0, 1, 1]),
            (50, [100, 3, 127, 128], [29, 4, 1, 1]), (50, [0, 0, 0], [rows, 1, 0]), (50, [5, 5], [rows + 1, 1]),
            (9, [0, 0], [2 ** 31 - 1, 2]), (9, [1, 2, 3], [2 ** 31 - 1] * 3), (9, [20, 20], [30, 1])):
        st = State(lengths, 8, 16, spare, rng, gpu)
        _step(st, counts, rows, gpu)
        _back(st, None, gpu)
    st = State([4, 5, 6], 2, 16, 9, rng, gpu)
    st.lengths[1] = -3
    st.t_lengths[1] = -3
    _step(st, [1, 1, 1], rows, gpu)


def test_no_rows(gpu):
    st = State([5, 0], 4, 16, 4, random.Random(0), gpu)
    assert _step(st, [0, 0], 0, gpu) == [5, 0]
    assert _step(st, [0, 1], 0, gpu) == [5, 0]


def test_counts_out_of_range_stay_in_bounds(gpu):
    """A count of held pages and of free ones beyond their arrays is taken as the array's end; giving back more pages than
    free_pages holds drops them."""
    st = State([20, 20], 4, 16, 3, random.Random(1), gpu)
    guard = torch.full((64,), 11, dtype=torch.int32, device=gpu)
    free = guard[16:16 + 5]
    free.copy_(_ints([1, 2, 3, 4, 5], gpu))
    held, count = _ints([99, -4], gpu), _ints([77], gpu)
    table = guard[32:40].view(2, 4)
    shadowkv.paged_reserve(st.t_lengths, _ints([10, 10], gpu), table, held, free, count, rows=20, page=16)
    assert count.item() == 3 and free.tolist() == [1, 2, 3, 4, 5]
    assert held.tolist() == [99, 2] and table.tolist() == [[11] * 4, [5, 4, 11, 11]]
    held.fill_(99)
    shadowkv.paged_release(st.t_lengths, _ints([0, 0], gpu), table, held, free, count, page=16)
    assert count.item() == 5 and held.tolist() == [0, 0] and st.t_lengths.tolist() == [0, 0]
    assert table.tolist() == [[-1] * 4] * 2
    assert guard.tolist() == [11] * 16 + free.tolist() + [11] * 11 + [-1] * 8 + [11] * 24


@pytest.mark.parametrize("B,most,page", [(1, 90, 16), (7, 400, 16), (30, 3000, 16), (1500, 60, 16), (64, 900, 256)])
def test_pages_that_do_not_exist_are_not_given_back(gpu, B, most, page):
    """Entries below zero among a sequence's pages (keys that no query sees) are no pages: those around them come back in
    their order, and what is reserved then has a place for every token."""
    rng = random.Random(B)
    lengths = [rng.randrange(1, most) for _ in range(B)]
    st = State(lengths, -(-most // page) + 2, page, 9, rng, gpu)
    for b in range(B):
        for i in range(st.held[b]):
            if rng.random() < (0.3 if b % 2 else 0.02) or b == i == 0:
                st.table[b][i] = rng.choice([-1, -2 ** 31])
    st.t_table.copy_(_ints(st.table, gpu))
    st.total -= sum(x < 0 for b in range(B) for x in st.table[b][:st.held[b]])
    for keep in ([rng.choice([-1, 0, n // 2, n]) for n in lengths], [0] * B):
        shadowkv.paged_release(st.t_lengths, _ints(keep, gpu), *st.args(), page=page)
        ref.release(st.lengths, keep, st.table, st.held, st.free, page)
        st.free = [p for p in st.free if p >= 0]
        st.check()
    assert len(st.free) == st.total
    totals = _step(st, [2] * B, 2 * B, gpu)
    assert sum(n == 2 for n in totals) == min(B, st.total)


def test_captured_step_follows_the_lengths(gpu):
    """A captured reserve with its advance, replayed beside eager work, gives what the lists give."""
    rng = random.Random(3)
    st = State([14, 0, 31], 16, 16, 30, rng, gpu)
    counts = _ints([1, 2, 1], gpu)
    out = {}

    def step():
        out["cu"], out["totals"], out["slots"] = shadowkv.paged_reserve(st.t_lengths, counts, *st.args(), rows=5, page=16)
        st.t_lengths.copy_(torch.maximum(st.t_lengths, out["totals"]))

    step()
    want = ref.reserve(st.lengths, [1, 2, 1], st.table, st.held, st.free, 5, 16)
    st.lengths = [max(n, t) for n, t in zip(st.lengths, want[1])]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with capture_graph(graph, gpu):
        step()
    for i in range(6):
        graph.replay()
        want = ref.reserve(st.lengths, [1, 2, 1], st.table, st.held, st.free, 5, 16)
        assert [out[x].tolist() for x in ("cu", "totals", "slots")] == list(want)
        st.lengths = [max(n, t) for n, t in zip(st.lengths, want[1])]
        st.check()
        if i == 3:
            _back(st, [2, -1, 0], gpu)


def _layout(P, H, page, order, gpu, gen):
    if order == "token":
        return [torch.randn(P, page, H, 128, generator=gen).to(BF16).to(gpu).transpose(1, 2) for _ in range(2)]
    if order == "pairs":  # keys and values in one tensor
        x = torch.randn(P, 2, H, page, 128, generator=gen).to(BF16).to(gpu)
        return [x[:, 0], x[:, 1]]
    if order == "slice":  # a layer of all, with room behind its rows
        x = torch.randn(2, 3, P, H, page, 136, generator=gen).to(BF16).to(gpu)
        return [x[0, 1, ..., :128], x[1, 1, ..., :128]]
    return [torch.randn(P, H, page, 128, generator=gen).to(BF16).to(gpu) for _ in range(2)]


@pytest.mark.parametrize("order", ["head", "token", "pairs", "slice"])
@pytest.mark.parametrize("N,H,page", [(1, 1, 16), (7, 3, 32), (300, 8, 64), (65, 2, 256)])
def test_write(gpu, order, N, H, page):
    """Each row in its place, to the bit (NaN too), and nothing else changed; slots outside the pages are dropped."""
    gen = torch.Generator().manual_seed(N * page)
    P = -(-N // page) + 3
    kp, vp = _layout(P, H, page, order, gpu, gen)
    qkv = torch.randn(N, 6 * H, 128, generator=gen).to(BF16)
    qkv[0, :, 3] = float("nan")
    qkv = qkv.to(gpu)
    k, v = qkv[:, 4 * H:5 * H], qkv[:, 5 * H:]
    slots = torch.randperm(P * page, generator=gen)[:N].to(torch.int32)
    bad = [-1, P * page, 2 ** 31 - 1, -2 ** 31, P * page + 5]
    for i in range(N // 6):
        slots[6 * i + 5] = bad[i % 5]
    want = [x.cpu().clone().view(torch.int16) for x in (kp, vp)]
    for r, s in enumerate(slots.tolist()):
        if 0 <= s < P * page:
            want[0][s // page, :, s % page] = k[r].cpu().view(torch.int16)
            want[1][s // page, :, s % page] = v[r].cpu().view(torch.int16)
    bases = [x._base if x._base is not None else x for x in (kp, vp)]
    sums = [x.cpu().clone() for x in bases]
    shadowkv.paged_write(k, v, kp, vp, slots.to(gpu))
    for x, w in zip((kp, vp), want):
        assert torch.equal(x.cpu().contiguous().view(torch.int16), w)
    if order == "slice":
        assert torch.equal(bases[0][..., 128:].cpu(), sums[0][..., 128:]) and torch.equal(bases[0][:, 0].cpu(),
                                                                                            sums[0][:, 0])


def test_write_other_rows(gpu):
    """Rows that cannot be read 16 bytes at a time, expanded rows, and none at all."""
    gen = torch.Generator().manual_seed(1)
    kp, vp = _layout(4, 2, 16, "head", gpu, gen)
    slots = torch.tensor([3, 40, 17], dtype=torch.int32, device=gpu)
    x = torch.randn(3, 2, 260, generator=gen).to(BF16).to(gpu)
    k, v = x[:, :, 1:129], x[:, :, 2:258:2]
    shadowkv.paged_write(k, v, kp, vp, slots)
    for r, s in enumerate(slots.tolist()):
        assert torch.equal(kp[s // 16, :, s % 16], k[r]) and torch.equal(vp[s // 16, :, s % 16], v[r])
    one = torch.randn(1, 1, 128, generator=gen).to(BF16).to(gpu).expand(3, 2, 128)
    shadowkv.paged_write(one, v, kp, vp, slots)
    for r, s in enumerate(slots.tolist()):
        assert torch.equal(kp[s // 16, :, s % 16], one[r])
    before = kp.clone()
    shadowkv.paged_write(k[:0], v[:0], kp, vp, slots[:0])
    assert torch.equal(kp, before)


def test_write_behind_2_to_the_31(gpu):
    """Elements past 2^31 and bytes past 2^32 of a pool."""
    P, H, page = (2 ** 31 // (8 * 256 * 128)) + 40, 8, 256
    kp, vp = (torch.empty(P, H, page, 128, dtype=BF16, device=gpu) for _ in range(2))
    gen = torch.Generator().manual_seed(2)
    k, v = (torch.randn(4, H, 128, generator=gen).to(BF16).to(gpu) for _ in range(2))
    at = [0, (P - 1) * page + 255, (P - 39) * page, (P // 2) * page + 3]
    for s in at:
        kp[s // page, :, s % page] = 0
    shadowkv.paged_write(k, v, kp, vp, torch.tensor(at, dtype=torch.int32, device=gpu))
    for r, s in enumerate(at):
        assert torch.equal(kp[s // page, :, s % page], k[r]) and torch.equal(vp[s // page, :, s % page], v[r])


def test_on_another_stream(gpu):
    gen = torch.Generator().manual_seed(4)
    kp, vp = _layout(8, 2, 16, "head", gpu, gen)
    k, v = (torch.randn(9, 2, 128, generator=gen).to(BF16).to(gpu) for _ in range(2))
    slots = torch.arange(30, 39, dtype=torch.int32, device=gpu)
    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        shadowkv.paged_write(k, v, kp, vp, slots)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(kp.transpose(1, 2).reshape(-1, 2, 128)[30:39], k)
