"""Whether an 8-bit cache's codes and scales share memory, without a GPU: against sets of bytes."""
import itertools
import random

import torch

from shadowkv_amd.kernels import shadowkv


def _runs(shape, strides, run, at):
    return [range(at + sum(i * s for i, s in zip(ix, strides)), at + sum(i * s for i, s in zip(ix, strides)) + run)
            for ix in itertools.product(*[range(n) for n in shape])]


def _bytes(shape, strides, run, at):
    return {x for r in _runs(shape, strides, run, at) for x in r}


def test_overlap_against_sets_of_bytes():
    """Layouts in any order of the axes with gaps between, at every distance around the places where they meet."""
    rng = random.Random(1)
    seen = {True: 0, False: 0}
    for _ in range(400):
        shape = tuple(rng.randint(1, 3) for _ in range(3))
        strides, extent = [0, 0, 0], 128
        for axis in rng.sample(range(3), 3):
            if shape[axis] > 1:
                strides[axis] = 16 * ((extent + 15) // 16 + rng.choice([0, 0, 1, 8, 20]))
                extent += (shape[axis] - 1) * strides[axis]
        blocks = rng.randint(1, 4)
        inner = rng.choice([0, 1])
        s_strides = [0, 0]
        if shape[inner] > 1:
            s_strides[inner] = blocks + rng.randint(0, 70)
        if shape[1 - inner] > 1:
            s_strides[1 - inner] = (shape[inner] - 1) * s_strides[inner] + blocks + rng.randint(0, 70)
        span = 4 * (blocks + sum((n - 1) * s for n, s in zip(shape, s_strides)))
        reach = lambda: rng.choice([-1, 1]) * 16 * rng.randint(0, extent // 16 + 20)  # noqa: E731
        v8, ks = reach(), rng.choice([4 * rng.randint(-span, (extent + span) // 2), 10 ** 6])
        vs = ks + rng.choice([4 * rng.randint(-span // 4 - 2, span // 4 + 2), span, 10 ** 7])
        parts = [_bytes(shape, strides, 128, 0), _bytes(shape, strides, 128, v8),
                 _bytes(shape[:2], [4 * s for s in s_strides], 4 * blocks, ks),
                 _bytes(shape[:2], [4 * s for s in s_strides], 4 * blocks, vs)]
        want = len(set().union(*parts)) < sum(map(len, parts))
        got = shadowkv._kv8_overlap(shape, tuple(strides), tuple(s_strides), blocks, v8, ks, vs)
        assert got == want, (shape, strides, s_strides, blocks, v8, ks, vs)
        seen[want] += 1
    assert min(seen.values()) > 40


def test_spans_of_a_layout():
    """The bytes from the first to the last of a layout's codes and scales, the room behind the scales left out."""
    codes, scale = torch.empty(2, 3, 100, 128, dtype=torch.float8_e4m3fn), torch.empty(2, 3, 9)
    layout = shadowkv._kv8_cache(codes, scale, "k8", 16)
    assert layout[3] == (codes.numel(), 4 * (5 * 9 + 7))
    side = torch.empty(2, 3, 100, 2, 128, dtype=torch.float8_e4m3fn)[:, :, :, 0]
    assert shadowkv._kv8_cache(side, scale, "k8", 16)[3][0] == 2 * codes.numel() - 128
    assert shadowkv._kv8_cache(codes[:, :1].expand(-1, 3, -1, -1), scale, "k8", 16)[3] is None
