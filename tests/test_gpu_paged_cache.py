"""The paged cache and its attention handler over whole sequences that begin, grow, are cut and end in shared pages;
against 64-bit restatements."""
import types

import pytest
import torch

from shadowkv_amd.models.attention import Cache2Attn
from shadowkv_amd.models.kvcache import method2kvcache
from shadowkv_amd.models.tensor_op import apply_rotary_pos_emb_cuda, build_cos_sin_cache
from shadowkv_amd.streams import capture_graph

from . import paged_reference as ref

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
L, HQ, H, D = 2, 8, 2, 128


def _made(gpu, B, max_length, **kw):
    config = types.SimpleNamespace(num_attention_heads=HQ, num_key_value_heads=H, hidden_size=HQ * D,
                                   num_hidden_layers=L)
    cache = method2kvcache["paged"](config, batch_size=B, max_length=max_length, device=gpu, **kw)
    table = build_cos_sin_cache(max_length, 500000.0, D, device=gpu)
    rope = lambda q, k, pos: tuple(  # noqa: E731
        apply_rotary_pos_emb_cuda(x, table, pos.unsqueeze(1).expand(-1, x.shape[1], -1)) for x in (q, k))
    return cache, Cache2Attn[type(cache)](cache, HQ // H, D, HQ * D, rope_f=rope), rope


def _inputs(B, T, g, gpu):
    """A projection's rows of one layer, as views [B, heads, T, 128]."""
    qkv = torch.randn(B, T, HQ + 2 * H, D, generator=g).to(BF16).to(gpu)
    return [x.transpose(1, 2).contiguous() for x in qkv.split((HQ, H, H), 2)]


class Model:
    """What each sequence was given, by layer, on the CPU."""

    def __init__(self, B):
        self.k = [[torch.zeros(H, 0, D) for _ in range(L)] for _ in range(B)]
        self.v = [[torch.zeros(H, 0, D) for _ in range(L)] for _ in range(B)]

    def add(self, b, layer, k, v):
        self.k[b][layer] = torch.cat([self.k[b][layer], k.cpu().double()], 1)
        self.v[b][layer] = torch.cat([self.v[b][layer], v.cpu().double()], 1)

    def cut(self, b, n):
        for x in (self.k[b], self.v[b]):
            x[:] = [y[:, :n] for y in x]

    def held(self):
        return [x[0].shape[1] for x in self.k]

    def check(self, b, layer, q, out, window):
        n = q.shape[0]
        ref.check(out, *ref.attention(q, self.k[b][layer], self.v[b][layer], n, window), bits=8)


def _packed_step(cache, attn, rope, model, counts, pad, g, gpu, window, served=None, max_new=None):
    """One step of packed rows through the layers, its outputs against the model's."""
    N = sum(counts) + pad
    held = model.held()
    pos = torch.cat([h + torch.arange(c) for h, c in zip(held, counts)] + [torch.zeros(pad)]).long().view(1, N).to(gpu)
    dev = torch.tensor(counts, dtype=torch.int32, device=gpu)
    for layer in range(L):
        q, k, v = _inputs(1, N, g, gpu)
        out = attn.prefill(q, k, v, pos, layer, counts=dev if layer == 0 else None, max_new=max_new)
        assert out.shape == (1, N, HQ, D)
        rq, rk = rope(q, k, pos)
        at = 0
        for b, c in enumerate(counts):
            rows = slice(at, at + c)
            at += c
            if served is not None and not served[b]:
                assert not out[0, rows].any()
            elif c:
                model.add(b, layer, rk[0, :, rows], v[0, :, rows])
                model.check(b, layer, rq[0, :, rows].transpose(0, 1), out[0, rows], window)
        assert not out[0, at:].any()
    assert cache.lengths.tolist() == model.held()
    if served is not None:
        assert cache.refused().tolist() == [not s and c > 0 for s, c in zip(served, counts)]


@pytest.mark.parametrize("page,window", [(16, None), (64, 50), (32, None)])
def test_sequences(gpu, page, window):
    """Prompts in pieces beside decoded tokens, drafts of which some are dropped, a sequence that ends and one that takes its
    place, a pool that runs out; all rows read back."""
    g = torch.Generator().manual_seed(page)
    B = 4
    cache, attn, rope = _made(gpu, B, 512, page=page, pages=-(-700 // page), window=window)
    for _ in range(2):  # (the second after clear(), over the first one's remains)
        model = Model(B)
        step = lambda counts, pad=0, **kw: _packed_step(cache, attn, rope, model, counts, pad, g, gpu, window, **kw)  # noqa
        step([130, 7, 1, 0], pad=5)
        step([1, 40, 1, 90], max_new=90)
        step([1, 1, 1, 1], max_new=1)
        step([3, 5, 2, 4], pad=2, max_new=5)
        keep = [134, 49, 5, 92]
        cache.trim(torch.tensor(keep, dtype=torch.int32, device=gpu), 134)
        for b, n in enumerate(keep):
            model.cut(b, n)
        step([1, 1, 1, 1], max_new=1)
        for T in (1, 3):  # T of each, [B, heads, T, 128]
            pos = torch.tensor(model.held()).unsqueeze(1) + torch.arange(T)
            for layer in range(L):
                q, k, v = _inputs(B, T, g, gpu)
                out = attn.decode(q, k, v, pos.to(gpu), layer)
                rq, rk = rope(q, k, pos.to(gpu))
                for b in range(B):
                    model.add(b, layer, rk[b], v[b])
                    model.check(b, layer, rq[b].transpose(0, 1), out[b], window)
        cache.trim(torch.where(torch.arange(B, device=gpu) == 0, 0, cache.lengths).to(torch.int32), max(model.held()[1:]))
        model.cut(0, 0)
        step([0, 1, 300, 300], served=[True, True, True, False], max_new=300)
        step([60, 1, 1, 0])
        for b in range(B):
            n = model.held()[b]
            for layer in range(L):
                if n:
                    got = cache.get_kv(layer, b, n)
                    assert torch.equal(got[0].cpu().double(), model.k[b][layer])
                    assert torch.equal(got[1].cpu().double(), model.v[b][layer])
        cache.clear()


def test_captured_steps(gpu):
    """Decode steps of one captured graph, replayed while sequences end and begin between them, give the eager bits."""
    g = torch.Generator().manual_seed(0)
    B, page = 3, 16
    made = [_made(gpu, B, 256, page=page, pages=30) for _ in range(2)]
    x = [_inputs(B, 1, g, gpu) for _ in range(L)]
    pos = torch.zeros(B, 1, dtype=torch.int64, device=gpu)
    prompt = _inputs(1, 90, g, gpu)
    counts = torch.tensor([60, 0, 30], dtype=torch.int32, device=gpu)
    outs = []
    for cache, attn, _ in made:
        for layer in range(L):
            attn.prefill(*prompt, torch.arange(90, device=gpu).view(1, 90), layer, counts=counts)

    def step(cache, attn):
        pos.copy_(cache.lengths.view(B, 1))
        return [attn.decode(*x[layer], pos, layer) for layer in range(L)]

    cache, attn, _ = made[0]
    step(cache, attn)
    step(*made[1][:2])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    before = cache.kv_offset
    with capture_graph(graph, gpu):
        outs = step(cache, attn)
    cache.kv_offset = before
    for i in range(20):
        for layer in range(L):
            for t in x[layer]:
                t.normal_()
        cache.check_capacity(1)
        graph.replay()
        cache.advance(1)
        want = step(*made[1][:2])
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)
        for name in ("lengths", "table", "held", "free_count"):
            assert torch.equal(getattr(cache, name), getattr(made[1][0], name)), name
        if i in (4, 11):
            for c, _, _ in made:
                keep = c.lengths.clone()
                keep[i % 3] = 0
                c.trim(keep, 256)
                c.kv_offset = 100 + i


def test_refused_follows_replays(gpu):
    """Of two captured steps and eager ones between them, refused() is the last one's that ran."""
    g = torch.Generator().manual_seed(1)
    B = 2
    cache, attn, _ = _made(gpu, B, 256, page=16, pages=4)
    steps = {}
    for T in (1, 20):
        x = [_inputs(B, T, g, gpu) for _ in range(L)]
        pos = torch.zeros(B, T, dtype=torch.int64, device=gpu)
        steps[T] = lambda x=x, pos=pos: [attn.decode(*x[layer], pos, layer) for layer in range(L)]
        steps[T]()
        cache.clear()
    torch.cuda.synchronize()
    graphs = {}
    for T in steps:
        graphs[T] = torch.cuda.CUDAGraph()
        with capture_graph(graphs[T], gpu):
            outs = steps[T]()  # noqa: F841
    cache.clear()
    lengths = [0, 0]
    # 4 pages of 16: 20 tokens of both take them all, the next 20 lack pages, single tokens fit until 32.
    for T, how, refused in ((20, "replay", 0), (20, "replay", 1), (1, "replay", 0), (20, "eager", 1), (1, "replay", 0),
                            (20, "replay", 1), (1, "eager", 0), (20, "replay", 1)):
        graphs[T].replay() if how == "replay" else steps[T]()
        torch.cuda.synchronize()
        lengths = [n + (0 if refused else T) for n in lengths]
        assert cache.refused().tolist() == [bool(refused)] * B and cache.lengths.tolist() == lengths, (T, how)
        cache.kv_offset, cache.unfinished = max(lengths), 0


def test_captured_packed_steps_follow_the_counts(gpu):
    """A captured step of packed rows, replayed while its counts change, stores and answers what an eager one does; a
    sequence with more new tokens than the host's bound is left as it is, answered with zeros and refused()."""
    g = torch.Generator().manual_seed(2)
    B, N, most = 3, 12, 5
    made = [_made(gpu, B, 256, page=16, pages=40) for _ in range(2)]
    x = [_inputs(1, N, g, gpu) for _ in range(L)]
    counts = torch.zeros(B, dtype=torch.int32, device=gpu)
    rows = torch.arange(N, device=gpu)

    def step(cache, attn):
        ends = counts.cumsum(0)
        b = torch.searchsorted(ends, rows, right=True).clamp(max=B - 1)
        pos = (cache.lengths[b] + rows - (ends - counts)[b]).clamp(0, 255).view(1, N)
        return [attn.prefill(*x[layer], pos, layer, counts=counts, max_new=most) for layer in range(L)]

    for cache, attn, _ in made:
        step(cache, attn)
        cache.clear()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with capture_graph(graph, gpu):
        outs = step(*made[0][:2])
    made[0][0].clear()
    lengths = [0] * B
    for now in ([5, 2, 3], [1, 1, 1], [0, 5, 5], [6, 2, 4], [1, 7, 4], [4, 4, 4], [0, 0, 12], [2, 1, 0]):
        counts.copy_(torch.tensor(now, dtype=torch.int32))
        for t in (t for layer in x for t in layer):
            t.normal_()
        graph.replay()
        want = step(*made[1][:2])
        torch.cuda.synchronize()
        over = [n > most for n in now]
        lengths = [n + (0 if o else c) for n, c, o in zip(lengths, now, over)]
        for a, b in zip(outs, want):
            assert torch.equal(a, b)
            for i, o in enumerate(over):
                mine = a[0, sum(now[:i]):sum(now[:i + 1])]
                assert not mine.any() if o else not len(mine) or mine.any()
        for cache, _, _ in made:
            assert cache.lengths.tolist() == lengths and cache.refused().tolist() == over, now
        for name in ("table", "held", "free_count", "start"):
            assert torch.equal(getattr(made[0][0], name), getattr(made[1][0], name)), name
        for b in range(B):
            for layer in range(L):
                for p, r in zip(made[0][0].get_kv(layer, b, lengths[b]), made[1][0].get_kv(layer, b, lengths[b])):
                    assert torch.equal(p, r)
        assert max(lengths) <= made[1][0].get_kv_len()
