"""The 8-bit cache where tokens are dropped again: drafts that are rejected, captured too, against a cache that never saw
them."""
import pytest
import torch

from shadowkv_amd.streams import capture_graph

from .test_gpu_kv8 import _check_attn
from .test_gpu_kv8_cache import L, _layer, _made, _say, _step_inputs

pytestmark = pytest.mark.gpu


def _ints(x, gpu):
    return torch.tensor(x, dtype=torch.int32, device=gpu)


def _run(attn, inputs, pos, counts=None):
    return [attn.decode(*inputs[layer], pos, layer, counts=counts) for layer in range(L)]


def _held(cache):
    """Codes and scales of what each sequence holds."""
    out = []
    for b, n in enumerate(cache.lengths.tolist()):
        out += [c[:, b, :, :n].contiguous().view(torch.uint8) for c in (cache.k8, cache.v8)]
        out += [s[:, b, :, :(n + cache.block - 1) // cache.block] for s in (cache.k_scale, cache.v_scale)]
    return out


@pytest.mark.parametrize("block,window,sinks", [(16, None, 0), (64, 70, 4)])
def test_rejected_drafts(gpu, block, window, sinks):
    """Five drafted tokens a step, of which each sequence keeps some; the rejected ones (smaller than the others, so that
    no scale grows for them) leave no trace: the same codes, scales and later attention, bit for bit."""
    _say(f"kv8 rejected drafts block={block}")
    g = torch.Generator().manual_seed(block)
    B, cap, T = 3, 160, 5
    (one, attn, rope), (other, attn2, _) = [_made(gpu, B, cap, block=block, window=window, sinks=sinks) for _ in range(2)]
    prompt = [_step_inputs(B, 40, g, gpu) for _ in range(L)]
    n = [40, 11, 33]
    pos = torch.arange(40, device=gpu).expand(B, -1)
    for c, a in ((one, attn), (other, attn2)):
        for layer in range(L):
            a.prefill(*prompt[layer], pos, layer, counts=_ints(n, gpu))
        c.trim(c.lengths, max(n))
        assert c.get_kv_len() == 40
    held = list(n)
    for step in range(8):
        keep = [(step + 2 * b) % (T + 1) for b in range(B)]
        drafts = [_step_inputs(B, T, g, gpu) for _ in range(L)]
        for q, k, v in drafts:
            for b in range(B):
                k[b, :, keep[b]:] *= 0.01
                v[b, :, keep[b]:] *= 0.01
        pos = torch.tensor(held, device=gpu).unsqueeze(1) + torch.arange(T, device=gpu)
        got = _run(attn, drafts, pos)
        for layer in range(L):
            rq, _ = rope(drafts[layer][0], drafts[layer][1], pos)
            _check_attn(rq, _layer(one, layer), [x + T for x in held], None, block, window, sinks, got=got[layer])
        held = [x + m for x, m in zip(held, keep)]
        one.trim(one.start + _ints(keep, gpu), max(held))
        want = _run(attn2, drafts, pos, _ints(keep, gpu))
        other.trim(other.lengths, max(held))
        assert one.lengths.tolist() == held == other.lengths.tolist() and one.get_kv_len() == max(held)
        for a, b in zip(_held(one), _held(other)):
            assert torch.equal(a, b)
    for layer in range(L):
        q, k, v = _step_inputs(B, 1, g, gpu)
        pos = torch.tensor(held, device=gpu).unsqueeze(1)
        assert torch.equal(attn.decode(q, k, v, pos, layer), attn2.decode(q, k, v, pos, layer))


def test_captured_drafts(gpu):
    """A step of drafted tokens and the dropping of the rejected ones in one graph, replayed with other tokens and other
    decisions: as the eager calls from the same state."""
    _say("kv8 captured drafts")
    g = torch.Generator().manual_seed(2)
    B, T = 2, 4
    cache, attn, _ = _made(gpu, B, 300)
    prompt = [_step_inputs(B, 100, g, gpu) for _ in range(L)]
    for layer in range(L):
        attn.prefill(*prompt[layer], torch.arange(100, device=gpu).expand(B, -1), layer, counts=_ints([100, 9], gpu))
    inputs, keep = [_step_inputs(B, T, g, gpu) for _ in range(L)], _ints([1, 3], gpu)
    state = (cache.k8.view(torch.uint8), cache.v8.view(torch.uint8), cache.k_scale, cache.v_scale, cache.lengths, cache.start)

    def step():
        pos = cache.lengths.long().unsqueeze(1) + torch.arange(T, device=gpu)
        out = _run(attn, inputs, pos)
        cache.trim(cache.start + keep, cache.max_length)
        return out

    before, at = [x.clone() for x in state], cache.kv_offset
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with capture_graph(graph, gpu):
        out = step()
    for x, y in zip(state, before):
        x.copy_(y)
    cache.kv_offset = at
    held = [100, 9]
    for kept in ([4, 0], [0, 2], [3, 3], [1, 4]):
        keep.copy_(_ints(kept, gpu))
        for x in [x for layer in inputs for x in layer]:
            x.copy_(torch.randn(x.shape, generator=g).to(x.dtype))
        before = [x.clone() for x in state]
        cache.check_capacity(T)
        graph.replay()
        replayed, after = [x.clone() for x in out], [x.clone() for x in state]
        for x, y in zip(state, before):
            x.copy_(y)
        want = step()
        held = [x + m for x, m in zip(held, kept)]
        cache.kv_offset = max(held)
        assert all(torch.equal(x, y) for x, y in zip(replayed, want))
        assert all(torch.equal(x.nan_to_num(), y.nan_to_num()) for x, y in zip(state, after))
        assert cache.lengths.tolist() == held
