"""The 8-bit cache and its attention handler over whole sequences: prompts of different lengths in pieces, single and
drafted tokens, captured steps, reading back; against 64-bit restatements."""
import types

import pytest
import torch

from shadowkv_amd.models.attention import Cache2Attn
from shadowkv_amd.models.kvcache import method2kvcache
from shadowkv_amd.models.tensor_op import apply_rotary_pos_emb_cuda, build_cos_sin_cache
from shadowkv_amd.streams import capture_graph

from .test_gpu_kv8 import _check_attn

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
L, HQ, H, D = 2, 8, 2, 128


def _say(msg):
    print(msg, flush=True)


def _made(gpu, B, max_length, **kw):
    config = types.SimpleNamespace(num_attention_heads=HQ, num_key_value_heads=H, hidden_size=HQ * D,
                                   num_hidden_layers=L)
    cache = method2kvcache["kv8"](config, batch_size=B, max_length=max_length, device=gpu, **kw)
    table = build_cos_sin_cache(max_length, 500000.0, D, device=gpu)
    rope = lambda q, k, pos: tuple(  # noqa: E731
        apply_rotary_pos_emb_cuda(x, table, pos.unsqueeze(1).expand(-1, x.shape[1], -1)) for x in (q, k))
    return cache, Cache2Attn[type(cache)](cache, HQ // H, D, HQ * D, rope_f=rope), rope


def _step_inputs(B, T, g, gpu):
    """A projection's rows of one layer, as views [B, heads, T, 128]."""
    qkv = torch.randn(B, T, HQ + 2 * H, D, generator=g).to(BF16).to(gpu)
    return [x.transpose(1, 2).contiguous() for x in qkv.split((HQ, H, H), 2)]


def _layer(cache, layer):
    return cache.k8[layer], cache.v8[layer], cache.k_scale[layer], cache.v_scale[layer]


@pytest.mark.parametrize("block,window,sinks", [(64, None, 0), (16, 50, 4), (128, 90, 0)])
def test_sequences(gpu, block, window, sinks):
    """Every step's attention over what the cache then holds, and the cache's rows against the ones that were given."""
    _say(f"kv8 cache block={block} window={window}")
    g = torch.Generator().manual_seed(block)
    B, cap = 3, 400
    cache, attn, rope = _made(gpu, B, cap, block=block, window=window, sinks=sinks)
    given = [[[], []] for _ in range(B)]  # of the last layer: keys and values by sequence, as they were written
    held = [0] * B
    steps = [(130, [130, 7, 1]), (40, [40, 0, 33]), (1, None), (1, None), (4, None), (9, [9, 1, 2]), (1, [1, 0, 1])]
    for turn in range(2):  # (the second after clear(), over the first one's remains)
        for T, counts in steps:
            n = counts or [T] * B
            pos = torch.tensor(held).unsqueeze(1) + torch.arange(T)
            for layer in range(L):
                q, k, v = _step_inputs(B, T, g, gpu)
                dev = None if counts is None else torch.tensor(counts, dtype=torch.int32, device=gpu)
                run = attn.prefill if T > 4 else attn.decode
                out = run(q, k, v, pos.to(gpu), layer, counts=dev)
                lengths = [a + b for a, b in zip(held, n)]
                rq, rk = rope(q, k, pos.to(gpu))
                _check_attn(rq, _layer(cache, layer), lengths, counts, block, window, sinks, got=out)
            for b in range(B):
                given[b][0].append(rk[b, :, :n[b]].cpu())
                given[b][1].append(v[b, :, :n[b]].cpu())
            held = lengths
            assert cache.lengths.tolist() == held
        assert cache.get_kv_len() == sum(T for T, _ in steps)
        cache.print_stats()
        cache.H2D()
        # A code is off by half a step, 2^-4 of the value or, where it is subnormal, 2^-10 of the scale; encoding again
        # under larger scales, by powers of two, adds at most as much again of the last scale's subnormal steps.
        for back, scale, which in zip(cache.get_kv(L - 1, 0, cap), (cache.k_scale, cache.v_scale), (0, 1)):
            for b in range(B):
                x = torch.cat(given[b][which], 1).double()
                got = back[b, :, :held[b]].cpu().double()
                s = scale[L - 1, b].cpu().double().repeat_interleave(block, 1)[:, :held[b], None]
                assert ((got - x).abs() <= x.abs() * 2.0 ** -4 + 3 * 2.0 ** -10 * s).all()
        cache.clear()
        given, held = [[[], []] for _ in range(B)], [0] * B
        assert cache.get_kv_len() == 0 and cache.lengths.tolist() == held


@pytest.mark.parametrize("window", [None, 64])
def test_captured_steps(gpu, window):
    """A whole step of both layers captured once and replayed while the lengths grow, with eager steps between the
    replays: every replay as the eager step from the same state."""
    _say(f"kv8 cache captured window={window}")
    g = torch.Generator().manual_seed(9)
    B, cap = 2, 1500
    cache, attn, _ = _made(gpu, B, cap, window=window)
    counts = torch.tensor([1300, 20], dtype=torch.int32, device=gpu)
    for layer in range(L):
        attn.prefill(*_step_inputs(B, 1300, g, gpu), torch.arange(1300, device=gpu).expand(B, -1), layer, counts=counts)
    inputs = [_step_inputs(B, 1, g, gpu) for _ in range(L)]
    pos = cache.lengths.long().unsqueeze(1)

    def step():
        return [attn.decode(*inputs[layer], pos, layer) for layer in range(L)]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    saved = cache.kv_offset
    with capture_graph(graph, gpu):
        out = step()
    cache.kv_offset = saved
    for _ in range(4):
        for layer in range(L):
            for x in inputs[layer]:
                x.copy_(torch.randn(x.shape, generator=g).to(BF16))
        pos.copy_(cache.lengths.long().unsqueeze(1))
        state = (cache.k8.view(torch.uint8), cache.v8.view(torch.uint8), cache.k_scale, cache.v_scale, cache.lengths)
        before = [x.clone() for x in state]
        cache.check_capacity(1)
        graph.replay()
        replayed = [x.clone() for x in out]
        after = [x.clone() for x in state]
        for x, y in zip(state, before):
            x.copy_(y)
        assert all(torch.equal(x, y) for x, y in zip(replayed, step()))
        assert all(torch.equal(x.nan_to_num(), y.nan_to_num()) for x, y in zip(state, after))
    assert cache.lengths.tolist() == [1305, 25]
