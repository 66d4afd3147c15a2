"""The 8-bit KV cache's operators (skv_kv8_write, skv_kv8_read, skv_kv8_attn) against 64-bit restatements."""
import math

import pytest
import torch

from shadowkv_amd.kernels import shadowkv
from shadowkv_amd.streams import capture_graph

pytestmark = pytest.mark.gpu
E4M3, BF16 = torch.float8_e4m3fn, torch.bfloat16
D = 128


def _say(msg):
    print(msg, flush=True)


def _bytes(t):
    return t.contiguous().view(torch.uint8)


def _same(a, b):
    """Equal values, NaN equal to NaN."""
    a, b = a.cpu().double(), b.cpu().double()
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


def _e4m3(x):
    """float64 -> the nearest e4m3 value, ties to even (|x| <= 464); NaN and infinities NaN."""
    step = torch.exp2(torch.frexp(x)[1].double() - 4).clamp(min=2.0 ** -9)
    return torch.where(x.isfinite(), torch.round(x / step) * step, torch.nan)


def _written(x, codes, scale, start, counts, block):
    """The write's definition, block by block, on CPU tensors in float64: the new codes' values and scales."""
    val, sc = codes.double(), scale.double()
    B, H, T, _ = x.shape
    cap = codes.shape[2]
    for b in range(B):
        st, n = int(start[b]), T if counts is None else min(max(int(counts[b]), 0), T)
        end = min(st + n, cap)
        if st < 0 or end <= st:
            continue
        for h in range(H):
            for j in range(st // block, (end - 1) // block + 1):
                lo, hi = max(st, j * block), min(end, (j + 1) * block)
                new = x[b, h, lo - st:hi - st].double()
                top = new[new.isfinite()].abs().max().item() if new.isfinite().any() else 0.0
                s = 2.0 ** -126
                if top > 0:
                    e = math.floor(math.log2(top)) - 10
                    while top > 448 * 2.0 ** e:
                        e += 1
                    s = 2.0 ** max(e, -126)
                if j * block < st:
                    was = sc[b, h, j].item()
                    if was >= s:
                        s = was
                    else:
                        val[b, h, j * block:st] = _e4m3(val[b, h, j * block:st] * (was / s))
                sc[b, h, j] = s
                val[b, h, lo:hi] = _e4m3(new / s)
    return val, sc


def _garbage(shape, gen):
    """Codes of every kind, NaN among them."""
    return torch.randint(0, 256, shape, generator=gen, dtype=torch.uint8).view(E4M3)


def _caches(B, H, cap, block, gen, gpu, order="bhs", extra=0):
    """k8, v8, k_scale, v_scale of garbage with garbage scales, in one of three layouts."""
    nb = (cap + block - 1) // block + extra
    out = []
    for _ in range(2):
        if order == "bsh":  # tokens outside heads
            c = _garbage((B, cap, H, D), gen).to(gpu).permute(0, 2, 1, 3)
        elif order == "slice":  # a layer of a larger buffer, with room behind its rows
            c = _garbage((B, H, cap + 3, D + 16), gen).to(gpu)[:, :, :cap, :D]
        else:
            c = _garbage((B, H, cap, D), gen).to(gpu)
        out.append(c)
    scales = [torch.exp2(torch.randint(-6, 7, (B, H, nb), generator=gen).float()).to(gpu) for _ in range(2)]
    return out + scales


def _rows(B, H, T, gen, gpu, spread=2.0):
    """Rows as a view of a projection's output, of very different sizes from token to token."""
    x = torch.randn(B, T, H, D, generator=gen) * torch.exp(spread * torch.randn(B, T, 1, 1, generator=gen))
    return x.to(BF16).to(gpu).transpose(1, 2)


def _check_write(k, v, caches, start, counts, block):
    k8, v8, ks, vs = caches
    before = [t.cpu().clone() for t in caches]
    shadowkv.kv8_write(k, v, k8, v8, ks, vs, torch.tensor(start, dtype=torch.int32, device=k.device),
                       counts=None if counts is None else torch.tensor(counts, dtype=torch.int32, device=k.device),
                       block=block)
    for x, codes, scale, c0, s0 in ((k, k8, ks, before[0], before[2]), (v, v8, vs, before[1], before[3])):
        val, sc = _written(x.cpu(), c0, s0, start, counts, block)
        assert torch.equal(scale.cpu().double(), sc)
        got = codes.cpu()
        assert _same(got, val)
        rewritten = torch.zeros(got.shape, dtype=torch.bool)
        for b, st in enumerate(start):
            n = x.shape[2] if counts is None else min(max(counts[b], 0), x.shape[2])
            if st >= 0 and n > 0 and st < got.shape[2]:
                rewritten[b, :, st // block * block:st + n] = True
        assert torch.equal(_bytes(got)[~rewritten], _bytes(c0)[~rewritten]), "a row that the call does not own changed"


@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("T,start,counts", [
    (1, [0, 5, 63], None), (1, [64, 127, 15], [1, 0, 1]), (3, [62, 126, 0], None), (17, [15, 0, 200], [17, 1, 9]),
    (130, [0, 1, 100], None), (200, [3, 64, 77], [200, 0, -4]), (65, [190, 255, 256], None),
    (9, [-1, 250, 300], [9, 12, 9])])
def test_write(gpu, block, T, start, counts):
    """Every code and scale equal to the definition's; blocks begun before, ends inside a block, rows past the
    capacity (256 tokens), counts of zero, below and above T, an inactive sequence."""
    _say(f"kv8_write block={block} T={T} start={start} counts={counts}")
    g = torch.Generator().manual_seed(block + T)
    B, H, cap = 3, 2, 256
    _check_write(_rows(B, H, T, g, gpu), _rows(B, H, T, g, gpu), _caches(B, H, cap, block, g, gpu), start, counts, block)


@pytest.mark.parametrize("order", ["bsh", "slice"])
def test_write_layouts(gpu, order):
    """Cache layouts other than [B, H, S, 128], scales with room behind, unaligned rows (copied), one kv head."""
    _say(f"kv8_write layout {order}")
    g = torch.Generator().manual_seed(3)
    for H in (1, 3):
        k = _rows(2, H, 40, g, gpu)
        v = torch.randn(2, H, 40, D + 1, generator=g).to(BF16).to(gpu)[..., 1:]
        _check_write(k, v, _caches(2, H, 100, 32, g, gpu, order, extra=2), [7, 61], None, 32)


def test_write_odd_values(gpu):
    """Zeros (scale 2^-126), bf16's smallest and largest magnitudes, infinities and NaN (both NaN, and left out of
    the scale), signed zeros, ties of the rounding, magnitudes at 448 times a power of two."""
    _say("kv8_write odd values")
    x = torch.zeros(1, 1, 7 * 16, D)
    x[0, 0, 16:32] = torch.tensor([2.0 ** -133, -2.0 ** -133, 2.0 ** -126, 0.0]).repeat(32)
    x[0, 0, 32:48] = torch.tensor([3.3895313892515355e38, -1.0, 2.0 ** 100, -3.3895313892515355e38]).repeat(32)
    x[0, 0, 48:64] = torch.tensor([math.inf, -math.inf, math.nan, 5.0]).repeat(32)
    x[0, 0, 64:80] = math.inf
    x[0, 0, 80:96] = torch.tensor([448.0, 17.0, 19.0, -25.0, 27.0, 2.0 ** -10, 3 * 2.0 ** -10, -0.0]).repeat(16)
    x[0, 0, 96:112] = torch.tensor([450.0, 1.0625, 1.1875, -1.3125]).repeat(32)
    x = x.to(BF16).to(gpu)
    g = torch.Generator().manual_seed(0)
    caches = _caches(1, 1, 112, 16, g, gpu)
    _check_write(x, -x, caches, [0], None, 16)
    assert torch.equal(caches[2].cpu()[0, 0, [0, 4, 5, 6]].log2(), torch.tensor([-126.0, -126.0, 0.0, 1.0]))
    assert caches[0][0, 0, 48:80].isnan().float().mean() == (0.75 + 1.0) / 2


def test_write_token_by_token(gpu):
    """Tokens appended one at a time, each larger than the last: the block's scale grows at every step, and its
    older rows are encoded again each time; a second, smaller pass over the same positions leaves scales alone."""
    _say("kv8_write token by token")
    g = torch.Generator().manual_seed(5)
    B, H, cap, block = 2, 2, 64, 32
    caches = _caches(B, H, cap, block, g, gpu)
    caches[2].fill_(2.0 ** -126)
    caches[3].fill_(2.0 ** -126)
    for t in range(40):
        k = (torch.randn(B, H, 1, D, generator=g) * 1.5 ** t).to(BF16).to(gpu)
        v = (torch.randn(B, H, 1, D, generator=g) * 1.5 ** (t % 7)).to(BF16).to(gpu)
        _check_write(k, v, caches, [t, t + 3], None, block)
    scales = [c.clone() for c in caches[2:]]
    small = (torch.randn(B, H, 1, D, generator=g) * 1e-3).to(BF16).to(gpu)
    _check_write(small, small, caches, [39, 42], None, block)
    assert all(torch.equal(a, b) for a, b in zip(scales, caches[2:]))


@pytest.mark.parametrize("block", [16, 64, 128])
def test_read(gpu, block):
    """Rows and chunks as bf16, exactly; chunks that pass the end, negative and far ids read as zeros; from
    layouts other than [B, H, S, 128] and from pinned host memory."""
    _say(f"kv8_read block={block}")
    g = torch.Generator().manual_seed(block)
    B, H, cap = 2, 3, 333
    for order in ("bhs", "bsh", "slice"):
        k8, _, ks, _ = _caches(B, H, cap, block, g, gpu, order)
        want = (k8.cpu().double() * ks.cpu().double().repeat_interleave(block, 2)[:, :, :cap, None]).to(BF16)
        for start, rows in ((0, cap), (17, 1), (100, 129), (332, 1)):
            got = shadowkv.kv8_read(k8, ks, start, rows, block=block)
            assert _same(got, want[:, :, start:start + rows])
        for chunk in (1, 8, 24):
            ids = torch.randint(0, cap // chunk + 1, (B, H, 21), generator=g)  # (the last chunk may pass the end)
            ids[0, 1, 3], ids[1, 2, 20], ids[0, 0, 0] = -1, 10 ** 12, cap // chunk + 1
            rows = (ids.unsqueeze(3) * chunk + torch.arange(chunk)).view(B, H, -1)
            inside = (rows >= 0) & (rows < cap)
            w = want.gather(2, rows.clamp(0, cap - 1).unsqueeze(3).expand(-1, -1, -1, D))
            w = torch.where(inside.unsqueeze(3), w, 0.0)
            got = shadowkv.kv8_read_chunks(k8, ks, ids.to(gpu), chunk, block=block)
            assert _same(got, w)
            if order == "bhs":
                host = torch.empty(k8.shape, dtype=E4M3, pin_memory=True)
                host.copy_(k8)
                assert torch.equal(_bytes(shadowkv.kv8_read_chunks(host, ks, ids.to(gpu), chunk, block=block)),
                                   _bytes(got))


def _filled(B, H, cap, block, gen, gpu, order="bhs"):
    """Caches of ordinary keys and values (blocks of different sizes), every token of the capacity."""
    caches = _caches(B, H, cap, block, gen, gpu, order)
    k = torch.randn(B, H, cap, D, generator=gen)
    v = torch.randn(B, H, cap, D, generator=gen) * torch.exp(torch.randn(B, 1, cap, 1, generator=gen)) + 0.3
    shadowkv.kv8_write(k.to(BF16).to(gpu), v.to(BF16).to(gpu), *caches, torch.zeros(B, dtype=torch.int32, device=gpu),
                       block=block)
    return caches


def _see(n, T, length, window, sinks):
    """[T, length] truth values: what each query sees."""
    p = length - n + torch.arange(T).unsqueeze(1)
    j = torch.arange(length).unsqueeze(0)
    see = (j <= p) & (torch.arange(T) < n).unsqueeze(1)
    return see if window is None else see & ((j > p - window) | (j < sinks))


def _check_attn(q, caches, lengths, counts, block, window=None, sinks=0, scale=None, got=None):
    """Tolerance: the output's rounding, 2^-8 of the value; and of the largest value seen: twice a score's error
    (130 fp32 roundings of the sum of the products' magnitudes, 2^-22 for the exponential), a probability's two parts
    (2^-15) and the fp32 sums over the keys (2^-24 a term, numerator and denominator)."""
    k8, v8, ks, vs = caches
    B, Hq, T, _ = q.shape
    H, cap = k8.shape[1], k8.shape[2]
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=q.device)  # noqa: E731
    if got is None:
        got = shadowkv.kv8_attn(q, *caches, ints(lengths), counts=None if counts is None else ints(counts), block=block,
                                window=window, sinks=sinks, scale=scale)
    assert got.shape == (B, T, Hq, D) and got.dtype == BF16 and got.is_contiguous()
    got = got.cpu().double()
    f = 1 / math.sqrt(D) if scale is None else scale
    wide = lambda s: s.cpu().double().repeat_interleave(block, 2)  # noqa: E731
    kd, vd, qd = k8.cpu().double(), v8.cpu().double(), q.cpu().double()
    kw, vw = wide(ks), wide(vs)
    for b in range(B):
        L = min(max(lengths[b], 0), cap)
        n = T if counts is None else min(max(counts[b], 0), T)
        see = _see(n, T, L, window, sinks)
        none = ~see.any(1)
        assert (got[b, none] == 0).all(), "rows that see nothing are zeros"
        if none.all():
            continue
        for hq in range(Hq):
            h = hq // (Hq // H)
            kk = kd[b, h, :L] * kw[b, h, :L, None]
            vv = vd[b, h, :L] * vw[b, h, :L, None]
            s = (f * qd[b, hq] @ kk.T).masked_fill(~see, -math.inf)
            w = torch.softmax(s, -1)
            clean = vv.nan_to_num(0.0)
            want = w @ clean
            want[(see.double() @ vv.isnan().double()) > 0] = math.nan
            want[none] = 0.0
            size = (abs(f) * qd[b, hq].abs() @ kk.nan_to_num(0.0).abs().T).masked_fill(~see, 0.0).amax(1)
            top = (see.unsqueeze(2) * clean.abs().unsqueeze(0)).amax((1, 2)) if T * L <= 40000 else clean.abs().max()
            tol = top * (2 * (130 * 2.0 ** -24 * size + 2.0 ** -22) + 2.0 ** -15 + 2 * L * 2.0 ** -24)
            g = got[b, :, hq]
            assert torch.equal(g.isnan(), want.isnan()), (b, hq)
            err = (g - want).abs().nan_to_num(0.0)
            lim = want.abs().nan_to_num(0.0) * 2.0 ** -8 + (tol.unsqueeze(1) if tol.dim() else tol)
            assert (err <= lim).all(), (b, hq, (err - lim).max(), err.max())


def _queries(B, Hq, T, gen, gpu, size=1.0):
    return (torch.randn(B, T, Hq, D, generator=gen) * size).to(BF16).to(gpu).transpose(1, 2)


@pytest.mark.parametrize("G", [1, 4, 7, 16])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("cap", [700, 2500])
def test_attn_one_token(gpu, G, block, cap):
    """Lengths from none to the whole capacity, around the groups of 32 keys and the chunks of 256 (a capacity that one
    workgroup takes, and one that is cut); everything behind a sequence's end is garbage (NaN codes and scales
    among it)."""
    _say(f"kv8_attn one token G={G} block={block} cap={cap}")
    g = torch.Generator().manual_seed(G * block)
    H = 2
    lengths = [0, 1, 15, 16, 31, 32, 33, 64, 129, 255, 256, 257, 300, 513, 699, 700, cap + 200, -3]
    caches = _filled(len(lengths), H, cap, block, g, gpu)
    for b, n in enumerate(lengths):
        n = max(n, 0)
        for c in caches[:2]:
            c.view(torch.uint8)[b, :, n:] = 0x7f
        for s in caches[2:]:
            s[b, :, (n + block - 1) // block:] = math.nan
    _check_attn(_queries(len(lengths), H * G, 1, g, gpu, 1.5), caches, lengths, None, block)
    _check_attn(_queries(len(lengths), H * G, 1, g, gpu, 1.5), caches, lengths, [1, 0] * 9, block)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (31, 4), (64, 0), (100, 33), (300, 64), (5000, 3), (200, 5000)])
@pytest.mark.parametrize("cap", [640, 2500])
def test_attn_one_token_window(gpu, window, sinks, cap):
    """Windows and sinks that begin and end inside a group, meet, and cover everything; hidden keys and values are
    NaN where a whole group or a part of one is hidden."""
    _say(f"kv8_attn one token window={window} sinks={sinks} cap={cap}")
    g = torch.Generator().manual_seed(window + sinks)
    H, G, block = 2, 4, 32
    lengths = [1, 30, 65, 99, 101, 333, 400, 401, 431, 639, 640]
    caches = _filled(len(lengths), H, cap, block, g, gpu)
    for b, n in enumerate(lengths):
        hidden = torch.zeros(cap, dtype=torch.bool)
        hidden[:n] = ~_see(1, 1, n, window, sinks)[0]
        hidden[n:] = True
        for c in caches[:2]:
            c.view(torch.uint8)[b, :, hidden.to(gpu)] = 0xff
    _check_attn(_queries(len(lengths), H * G, 1, g, gpu, 1.5), caches, lengths, None, block, window, sinks)


@pytest.mark.parametrize("H,G,T", [(2, 4, 2), (1, 1, 33), (3, 7, 19), (2, 17, 1), (1, 40, 1), (2, 16, 9), (8, 4, 70),
                                   (1, 4, 300)])
@pytest.mark.parametrize("block", [16, 128])
@pytest.mark.parametrize("cap", [450, 2500])
def test_attn_many(gpu, H, G, T, block, cap):
    """Several tokens, or more than 16 heads a kv head: rows around the tiles of 32 and 128, lengths around the
    tiles of 64 and shorter than the new tokens, ragged counts; garbage behind the ends."""
    _say(f"kv8_attn many H={H} G={G} T={T} block={block} cap={cap}")
    g = torch.Generator().manual_seed(H * G + T)
    lengths = [T, T + 1, 0, 64, 65, 191, 450, max(1, T // 2), 3000]
    counts = [T, max(1, T - 1), 1, T, T // 2, T, 0, T, T + 5]
    caches = _filled(len(lengths), H, cap, block, g, gpu, "bsh" if T == 19 else "bhs")
    for b, n in enumerate(lengths):
        for c in caches[:2]:
            c.view(torch.uint8)[b, :, n:] = 0x7f
        for s in caches[2:]:
            s[b, :, (n + block - 1) // block:] = math.inf
    q = _queries(len(lengths), H * G, T, g, gpu, 1.5)
    _check_attn(q, caches, lengths, counts, block)
    _check_attn(q, caches, lengths, None, block)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 2), (63, 1), (64, 64), (100, 33), (130, 0), (4000, 7), (90, 4000)])
@pytest.mark.parametrize("T,cap", [(5, 700), (5, 2500), (150, 700)])
def test_attn_many_window(gpu, window, sinks, T, cap):
    """Windows with sinks over several tokens, each with its own end."""
    _say(f"kv8_attn many window={window} sinks={sinks} T={T} cap={cap}")
    g = torch.Generator().manual_seed(window + sinks + T)
    lengths, counts = [T, 333, 700, 640, 65, 700], [T, T, T, T // 2, 1, max(1, T - 3)]
    caches = _filled(len(lengths), 2, cap, 64, g, gpu)
    q = _queries(len(lengths), 8, T, g, gpu, 1.5)
    _check_attn(q, caches, lengths, counts, 64, window, sinks)


@pytest.mark.parametrize("T,cap", [(1, 320), (2, 320), (2, 2500), (6, 2500), (70, 320)])
def test_attn_nan_where_seen_and_hidden(gpu, T, cap):
    """A NaN among the keys makes the rows that see it NaN, one among the values the dims of the rows that see it,
    and neither reaches a row that does not (a later key, or one behind the window)."""
    _say(f"kv8_attn NaN T={T} cap={cap}")
    g = torch.Generator().manual_seed(T)
    lengths = [300, 300, 299]
    for window, sinks in ((None, 0), (40, 10)):
        caches = _filled(3, 2, cap, 32, g, gpu)
        v8, k8 = caches[1].view(torch.uint8), caches[0].view(torch.uint8)
        v8[0, 0, 299, 5] = v8[0, 1, 270, 9] = v8[0, 1, 3, 127] = 0x7f
        v8[1, 0, 250, 64:70] = 0xff
        v8[2, 0, 200:260, 17] = 0x7f
        q = _queries(3, 8, T, g, gpu)
        _check_attn(q, caches, lengths, None, 32, window, sinks)
        k8[1, 1, 290, 3] = 0x7f
        got = shadowkv.kv8_attn(q, *caches, torch.tensor(lengths, dtype=torch.int32, device=gpu), block=32,
                                window=window, sinks=sinks).cpu()
        see = _see(T, T, 300, window, sinks)[:, 290]
        assert torch.equal(got[1, :, 4:].isnan().all(-1), see.unsqueeze(1).expand(T, 4))
        assert torch.equal(got[1, :, 4:].isnan().any(-1), see.unsqueeze(1).expand(T, 4))


@pytest.mark.parametrize("T,cap", [(3, 128), (3, 2500), (45, 128)])
def test_attn_padding_beside_nan(gpu, T, cap):
    """Padding rows are zeros where the sequence's own rows are NaN, and where their queries are NaN or infinite."""
    _say(f"kv8_attn padding beside NaN T={T} cap={cap}")
    g = torch.Generator().manual_seed(T)
    caches = _filled(2, 2, cap, 32, g, gpu)
    caches[1].view(torch.uint8)[:, :, 60] = 0x7f
    q = _queries(2, 8, T, g, gpu)
    q[:, :, T - 1] = math.nan
    q[0, :, T - 1] = math.inf
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    got = shadowkv.kv8_attn(q, *caches, ints([100, 61]), counts=ints([T - 1, 1]), block=32)
    sees = _see(T - 1, T, 100, None, 0)[:T - 1, 60].to(gpu)  # (the last queries of the 99 positions before)
    assert torch.equal(got[0, :T - 1].isnan().all(-1), sees.unsqueeze(1).expand(-1, 8)) and got[1, :1].isnan().all()
    assert not got[0, :T - 1][~sees].isnan().any()
    assert (got[0, T - 1:] == 0).all() and (got[1, 1:] == 0).all()


@pytest.mark.parametrize("T", [1, 40])
def test_attn_scores_of_every_size(gpu, T):
    """Scores that grow along the keys (the running maximum moves in every tile), that fall, and all-equal ones;
    a scale given; scales of the cache that differ by 2^30 from block to block."""
    _say(f"kv8_attn score sizes T={T}")
    g = torch.Generator().manual_seed(T + 1)
    L = 400
    for sign in (1.0, -1.0, 0.0):
        k = torch.linspace(-12, 12, L)[None, None, :, None] * sign + 0.1 * torch.randn(1, 1, L, D, generator=g)
        v = torch.randn(1, 1, L, D, generator=g) * torch.exp2(15.0 * torch.randint(-1, 2, (L // 16, 1), generator=g)
                                                              .expand(L // 16, 16).reshape(1, 1, L, 1))
        caches = _caches(1, 1, L, 16, g, gpu)
        shadowkv.kv8_write(k.to(BF16).to(gpu), v.to(BF16).to(gpu), *caches,
                           torch.zeros(1, dtype=torch.int32, device=gpu), block=16)
        q = torch.ones(1, 4, T, D).to(BF16).to(gpu)
        _check_attn(q, caches, [L], None, 16)
        _check_attn(q, caches, [L], None, 16, scale=0.01)


@pytest.mark.parametrize("T,cap", [(1, 320), (7, 320), (1, 2500), (7, 2500), (70, 320), (70, 2500)])
def test_attn_scales_that_are_hidden(gpu, T, cap):
    """Scales of blocks that a query does not see, behind its window or past the sequence's end, may be anything, and
    so may the codes there; a query that does see a block of NaN scales is NaN."""
    _say(f"kv8_attn hidden scales T={T} cap={cap}")
    g = torch.Generator().manual_seed(T + cap)
    odd = [math.nan, math.inf, -math.inf, -1.0]
    lengths, window, sinks = [300, 231], 30, 5
    for which in range(4):
        caches = _filled(2, 2, cap, 16, g, gpu)
        want = [c.clone() for c in caches]
        for b, L in enumerate(lengths):
            first = max(0, L - T - window + 1) // 16  # (the sinks' block is seen)
            for c, ones in zip(caches, want):
                if c.dtype == E4M3:
                    for x in (c, ones):
                        x.view(torch.uint8)[b, :, L:] = 0x7f
                        x.view(torch.uint8)[b, :, 16:16 * first] = 0x7f
                else:
                    c[b, :, 1:first] = odd[which]
                    c[b, :, (L - 1) // 16 + 1:] = odd[which]
                    ones[b, :, 1:first] = 1.0
        q = _queries(2, 8, T, g, gpu)
        at = torch.tensor(lengths, dtype=torch.int32, device=gpu)
        got = shadowkv.kv8_attn(q, *caches, at, block=16, window=window, sinks=sinks)
        _check_attn(q, want, lengths, None, 16, window, sinks, got=got)
        # seen by the first queries and not by the last ones (from T = 17 on)
        caches = _filled(2, 2, cap, 16, g, gpu)
        caches[2 + which % 2][:, :, (231 - T - 14) // 16] = math.nan
        got = shadowkv.kv8_attn(q, *caches, at, block=16, window=window, sinks=sinks).cpu()
        for b, L in enumerate(lengths):
            j = torch.arange(L) // 16 == (231 - T - 14) // 16
            hit = _see(T, T, L, window, sinks)[:, j].any(1)
            assert hit.any() or b == 0
            assert torch.equal(got[b].isnan().all(-1), hit.unsqueeze(1).expand(T, 8)), (which, b)
            assert torch.equal(got[b].isnan().any(-1), hit.unsqueeze(1).expand(T, 8)), (which, b)


@pytest.mark.parametrize("T", [1, 12, 50])
def test_attn_any_scales(gpu, T):
    """Scales that no write makes (no powers of two, zeros) and factors of the scores that are zero or negative."""
    _say(f"kv8_attn any scales T={T}")
    g = torch.Generator().manual_seed(T)
    caches = _filled(2, 2, 400, 32, g, gpu)
    q = _queries(2, 8, T, g, gpu)
    for factor in (0.0, -0.05, 0.3):
        _check_attn(q, caches, [400, 333], None, 32, scale=factor)
    for s in caches[2:]:
        s.mul_((0.6 + torch.rand(s.shape, generator=g)).to(gpu))
    caches[3][0, 1, 2] = 0.0
    caches[2][1, 0, 3] = 0.0
    _check_attn(q, caches, [400, 333], None, 32)
    _check_attn(q, caches, [400, 333], [T, T // 2], 32, 100, 40)


def test_attn_layouts(gpu):
    """Queries and caches of other strides: heads and tokens in any order, a key and its value side by side, one kv
    head's cache for all, a capacity of one, rows that start off 16 bytes."""
    _say("kv8_attn layouts")
    g = torch.Generator().manual_seed(21)
    for T in (1, 6, 45):
        for order in ("bsh", "slice"):
            _check_attn(_queries(2, 6, T, g, gpu), _filled(2, 3, 333, 16, g, gpu, order), [333, 150], None, 16)
        side = _garbage((2, 3, 200, 2, D), g).to(gpu)
        scales = torch.ones(2, 3, 7, 2, device=gpu)
        caches = [side[:, :, :, 0], side[:, :, :, 1], scales[..., 0].contiguous(), scales[..., 1].contiguous()]
        k, v = _rows(2, 3, 200, g, gpu, 0.3), _rows(2, 3, 200, g, gpu, 0.3)
        shadowkv.kv8_write(k, v, *caches, torch.zeros(2, dtype=torch.int32, device=gpu), block=32)
        _check_attn(_queries(2, 6, T, g, gpu), caches, [200, 64], None, 32)
        one = [c[:, :1].expand(-1, 3, *[-1] * (c.dim() - 2)) for c in caches]
        _check_attn(_queries(2, 6, T, g, gpu), one, [200, 64], None, 32)
        flat = torch.randn(2 * 6 * T * D + 1, generator=g).to(BF16).to(gpu)[1:].view(2, 6, T, D)
        _check_attn(flat, caches, [200, 64], None, 32)
        _check_attn(_queries(2, 6, T, g, gpu), _filled(2, 3, 1, 16, g, gpu), [1, 0], None, 16)


@pytest.mark.parametrize("H,G,T", [(2, 4, 33), (2, 16, 9), (1, 16, 40), (1, 4, 150)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (2700, 0), (2600, 70), (3500, 1000)])
def test_attn_many_on_long_caches(gpu, H, G, T, window, sinks):
    """Rows beyond a workgroup of 128 on caches of thousands of keys: several shares of them, waves with no rows, the
    ends of windows, padding, scales and layouts as elsewhere."""
    _say(f"kv8_attn many long H={H} G={G} T={T} window={window}")
    g = torch.Generator().manual_seed(T + G)
    caches = _filled(2, H, 4500, 32, g, gpu, "bsh" if T == 33 else "bhs")
    q = _queries(2, H * G, T, g, gpu)
    _check_attn(q, caches, [4500, 2811], None, 32, window, sinks)
    _check_attn(q, caches, [4433, T - 3], [T, T - 2], 32, window, sinks)
    _check_attn(q, caches, [3001, 0], [1, T], 32, window, sinks)


@pytest.mark.parametrize("window,sinks", [(None, 0), (2600, 10)])
def test_attn_many_on_long_caches_odd(gpu, window, sinks):
    """NaN and scales that no f16 holds together, among many rows on a long cache: seen by some, hidden from others."""
    _say(f"kv8_attn many long odd window={window}")
    g = torch.Generator().manual_seed(3)
    caches = _filled(2, 2, 4000, 16, g, gpu)
    q = _queries(2, 8, 50, g, gpu)
    v8 = caches[1].view(torch.uint8)
    v8[0, 0, 3960, 5] = v8[0, 1, 1375, 9] = v8[0, 1, 3, 127] = v8[0, 1, 2000, 64] = 0x7f
    v8[1, 0, 3970:3980, 64:70] = 0xff
    _check_attn(q, caches, [4000, 3990], None, 16, window, sinks)
    caches = _filled(2, 2, 4000, 16, g, gpu)
    caches[3].mul_(torch.exp2(torch.randint(-9, 9, caches[3].shape, generator=g).float()).to(gpu))
    _check_attn(q, caches, [4000, 3977], None, 16, window, sinks)
    caches[3].mul_((0.6 + torch.rand(caches[3].shape, generator=g)).to(gpu))
    _check_attn(q, caches, [4000, 3977], [50, 31], 16, window, sinks)
    caches[2][:, :, 3965 // 16] = math.nan  # seen by the last queries only
    caches[3][:, :, 1330 // 16] = math.nan  # with the window, by the first ones only
    got = shadowkv.kv8_attn(q, *caches, torch.tensor([4000, 3990], dtype=torch.int32, device=gpu), block=16,
                            window=window, sinks=sinks).cpu()
    for b, L in enumerate((4000, 3990)):
        j = torch.arange(L) // 16
        hit = _see(50, 50, L, window, sinks)[:, (j == 3965 // 16) | (j == 1330 // 16)].any(1)
        assert torch.equal(got[b].isnan().all(-1), hit.unsqueeze(1).expand(50, 8))
        assert torch.equal(got[b].isnan().any(-1), hit.unsqueeze(1).expand(50, 8))


@pytest.mark.parametrize("window,sinks", [(None, 0), (6800, 0), (6790, 70)])
def test_attn_many_rows_of_many_heads(gpu, window, sinks):
    """Enough workgroups of more than 128 rows, over shares of a long cache, for every CU (they are then larger): ends
    of windows, waves with no rows, padding, NaN seen by some, scales of any size, hidden ones of NaN."""
    _say(f"kv8_attn many rows and heads window={window}")
    g = torch.Generator().manual_seed(17)
    B, H, G, T, cap, block = 2, 8, 4, 33, 8000, 16
    q = _queries(B, H * G, T, g, gpu)
    caches = _filled(B, H, cap, block, g, gpu)
    _check_attn(q, caches, [8000, 4811], None, block, window, sinks)
    _check_attn(q, caches, [7933, 20], [T, 7], block, window, sinks)
    _check_attn(q, caches, [7001, 0], [1, T], block, window, sinks)
    v8 = caches[1].view(torch.uint8)
    v8[0, 0, 7975, 5] = v8[0, 1, 1190, 9] = v8[0, 2, 3, 127] = v8[0, 3, 5000, 64] = 0x7f
    v8[1, 0, 7980:7990, 64:70] = 0xff
    _check_attn(q, caches, [8000, 7999], None, block, window, sinks)
    caches = _filled(B, H, cap, block, g, gpu)
    caches[3].mul_(torch.exp2(torch.randint(-9, 9, caches[3].shape, generator=g).float()).to(gpu))
    caches[2].mul_((0.6 + torch.rand(caches[2].shape, generator=g)).to(gpu))
    _check_attn(q, caches, [8000, 7977], None, block, window, sinks)
    lengths = [8000, 7990]
    caches[2][:, :, 7975 // block] = math.nan  # seen by the last queries only
    caches[3][:, :, 1185 // block] = math.nan  # with a window, by the first ones only
    got = shadowkv.kv8_attn(q, *caches, torch.tensor(lengths, dtype=torch.int32, device=gpu), block=block,
                            window=window, sinks=sinks).cpu()
    for b, L in enumerate(lengths):
        j = torch.arange(L) // block
        hit = _see(T, T, L, window, sinks)[:, (j == 7975 // block) | (j == 1185 // block)].any(1)
        assert torch.equal(got[b].isnan().all(-1), hit.unsqueeze(1).expand(T, H * G))
        assert torch.equal(got[b].isnan().any(-1), hit.unsqueeze(1).expand(T, H * G))


def test_attn_long_and_uneven(gpu):
    """A batch of one long and many short sequences (chunks of several groups to a wave, 70 sequences over two
    passes of the plan), and a few tokens of long ones (keys split over workgroups)."""
    _say("kv8_attn long")
    g = torch.Generator().manual_seed(11)
    lengths = [20000] + [(37 * i) % 900 for i in range(69)]
    caches = _filled(70, 1, 20000, 64, g, gpu)
    _check_attn(_queries(70, 4, 1, g, gpu), caches, lengths, None, 64)
    _check_attn(_queries(70, 4, 3, g, gpu), caches, lengths, None, 64, 7000, 70)
    one = [c[:1] for c in caches]
    _check_attn(_queries(1, 4, 6, g, gpu), one, [19999], [5], 64)


def test_offsets_past_32_bits(gpu):
    """A head of 17.5 million tokens (2.24 GB of keys): rows written, read and attended to behind byte 2^31."""
    _say("kv8 offsets past 2^31")
    cap, block = 17_500_032, 64
    g = torch.Generator().manual_seed(2)
    caches = [torch.zeros(1, 1, cap, D, dtype=E4M3, device=gpu) for _ in range(2)] + \
        [torch.full((1, 1, cap // block), 2.0 ** -126, device=gpu) for _ in range(2)]
    start = 17_400_000
    k, v = _rows(1, 1, 500, g, gpu, 0.2), _rows(1, 1, 500, g, gpu, 0.2)
    at = torch.tensor([start], dtype=torch.int32, device=gpu)
    shadowkv.kv8_write(k, v, *caches, at, block=block)
    got = shadowkv.kv8_read(caches[0], caches[2], start, 500, block=block)
    assert (got.float() - k.float()).abs().max() <= k.float().abs().max() * 2 ** -3
    assert shadowkv.kv8_read(caches[0], caches[2], start - 100, 100, block=block).abs().max() == 0
    small = [c[:, :, start:start + 512].contiguous() for c in caches[:2]] + \
        [c[:, :, start // block:start // block + 8].contiguous() for c in caches[2:]]
    assert start % block == 0
    for T in (1, 9):
        q = _queries(1, 4, T, g, gpu)
        far = shadowkv.kv8_attn(q, *caches, at + 500, block=block, window=400)
        _check_attn(q, small, [500], None, block, window=400, got=far)


def test_captured_steps_follow_the_device(gpu):
    """Write and attention of a token, and of a few, captured once and replayed while the lengths grow on the
    device, two graphs in turn with eager work between them: every replay as the eager calls."""
    _say("kv8 captured")
    g = torch.Generator().manual_seed(8)
    B, H, G, block, cap = 3, 2, 4, 32, 2000
    caches = _filled(B, H, cap, block, g, gpu)
    pos = torch.tensor([5, 300, 1800], dtype=torch.int32, device=gpu)
    state = {}
    for T in (1, 4):
        k, v, q = _rows(B, H, T, g, gpu), _rows(B, H, T, g, gpu), _queries(B, H * G, T, g, gpu)

        def step(k=k, v=v, q=q, T=T):
            shadowkv.kv8_write(k, v, *caches, pos, block=block)
            return shadowkv.kv8_attn(q, *caches, pos + T, block=block, window=700, sinks=5)

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with capture_graph(graph, gpu):
            out = step()
        state[T] = (graph, out, k, v, q, step)
    for i in range(4):
        for T, (graph, out, k, v, q, step) in state.items():
            for x in (k, v, q):
                x.copy_(torch.randn(x.shape, generator=g).to(BF16))
            saved = [c.clone() for c in caches]
            graph.replay()
            replayed = out.clone()
            after = [c.clone() for c in caches]
            for c, s in zip(caches, saved):
                c.view(torch.uint8).copy_(s.view(torch.uint8))
            want = step()
            assert torch.equal(replayed, want)
            assert all(torch.equal(_bytes(a), _bytes(c)) for a, c in zip(after, caches))
            pos.add_(T)


def test_captured_prompt_pieces(gpu):
    """Many rows captured with their shares of a long cache by three graphs that are replayed in turn, with
    eager calls between: lengths and counts are read at each replay."""
    _say("kv8 captured pieces")
    g = torch.Generator().manual_seed(14)
    caches = _filled(2, 2, 5000, 64, g, gpu)
    lengths = torch.tensor([100, 5000], dtype=torch.int32, device=gpu)
    counts = torch.tensor([40, 40], dtype=torch.int32, device=gpu)
    runs = []
    for T, window in ((40, None), (13, 2800), (3, None)):
        q = _queries(2, 8, T, g, gpu)
        call = lambda q=q, window=window: shadowkv.kv8_attn(q, *caches, lengths, counts, block=64,  # noqa: E731
                                                            window=window)
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with capture_graph(graph, gpu):
            out = call()
        runs.append((graph, out, q, window, call))
    for L, n in (([5000, 37], [40, 2]), ([0, 4999], [1, 13]), ([3000, 2999], [0, 40]), ([5000, 5000], [13, 40])):
        lengths.copy_(torch.tensor(L, dtype=torch.int32))
        counts.copy_(torch.tensor(n, dtype=torch.int32))
        for graph, out, q, window, call in runs:
            graph.replay()
            got = out.clone()
            assert torch.equal(got, call())
            _check_attn(q, caches, L, n, 64, window, got=got)


def test_other_stream_and_repeats(gpu):
    """Calls on another stream than the default one, two at once, the same call twice: the same bits."""
    _say("kv8 streams")
    g = torch.Generator().manual_seed(4)
    caches = _filled(2, 2, 3000, 64, g, gpu)
    lengths = torch.tensor([3000, 2777], dtype=torch.int32, device=gpu)
    q1, q2 = _queries(2, 8, 1, g, gpu), _queries(2, 8, 40, g, gpu)
    want = [shadowkv.kv8_attn(q, *caches, lengths, block=64) for q in (q1, q2)]
    torch.cuda.synchronize()
    from shadowkv_amd.streams import side_stream
    got = []
    for role in ("fetch", "rebuild"):
        with torch.cuda.stream(side_stream(gpu, role)):
            got.append([shadowkv.kv8_attn(q, *caches, lengths, block=64) for q in (q1, q2)])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for pair in got for a, b in zip(pair, want))


def test_refusals(gpu):
    """Arguments that a call cannot serve are errors before any launch."""
    _say("kv8 refusals")
    g = torch.Generator().manual_seed(1)
    k8, v8, ks, vs = caches = _caches(2, 2, 64, 32, g, gpu)
    k, q = _rows(2, 2, 3, g, gpu), _queries(2, 4, 3, g, gpu)
    at = torch.zeros(2, dtype=torch.int32, device=gpu)

    def no(f, *a, **kw):
        with pytest.raises((ValueError, RuntimeError)):
            f(*a, **kw)

    for block in (0, 8, 48, 256, -16):
        no(shadowkv.kv8_write, k, k, *caches, at, block=block)
        no(shadowkv.kv8_attn, q, *caches, at, block=block)
        no(shadowkv.kv8_read, k8, ks, 0, 4, block=block)
    no(shadowkv.kv8_write, k, k, *caches, at, block=16)  # too few scales
    no(shadowkv.kv8_write, k, k, k8, k8, ks, vs, at, block=32)
    no(shadowkv.kv8_write, k, k, k8[:, :1].expand(-1, 2, -1, -1), v8[:, :1].expand(-1, 2, -1, -1), ks, vs, at, block=32)
    no(shadowkv.kv8_write, k.float(), k, *caches, at, block=32)
    no(shadowkv.kv8_write, k[:, :1], k[:, :1], *caches, at, block=32)
    no(shadowkv.kv8_write, k[:, :, :0], k[:, :, :0], *caches, at, block=32)
    no(shadowkv.kv8_write, k[..., :64], k[..., :64], *caches, at, block=32)
    no(shadowkv.kv8_write, k, k, k8.view(torch.uint8), v8, ks, vs, at, block=32)
    no(shadowkv.kv8_write, k, k, k8.cpu(), v8, ks, vs, at, block=32)
    no(shadowkv.kv8_write, k, k, k8, v8, ks.double(), vs, at, block=32)
    no(shadowkv.kv8_write, k, k, *caches, at.long(), block=32)
    no(shadowkv.kv8_write, k, k, *caches, at.cpu(), block=32)
    no(shadowkv.kv8_write, k, k, *caches, at[:1], block=32)
    no(shadowkv.kv8_write, k.clone().requires_grad_(), k, *caches, at, block=32)
    no(shadowkv.kv8_attn, q.clone().requires_grad_(), *caches, at, block=32)
    no(shadowkv.kv8_attn, _queries(2, 3, 1, g, gpu), *caches, at, block=32)
    no(shadowkv.kv8_attn, q, *caches, at, block=32, window=0)
    no(shadowkv.kv8_attn, q, *caches, at, block=32, sinks=4)
    no(shadowkv.kv8_attn, q, *caches, at, block=32, window=4, sinks=-1)
    no(shadowkv.kv8_attn, q, *caches, at, counts=at[:1], block=32)
    no(shadowkv.kv8_attn, q, k8, v8[:, :, :32], ks, vs, at, block=32)
    no(shadowkv.kv8_read, k8, ks, 0, 65, block=32)
    no(shadowkv.kv8_read, k8, ks, -1, 4, block=32)
    no(shadowkv.kv8_read, k8, ks, 0, 0, block=32)
    no(shadowkv.kv8_read, k8.cpu(), ks, 0, 4, block=32)  # not pinned
    ids = torch.zeros(2, 2, 4, dtype=torch.int64, device=gpu)
    no(shadowkv.kv8_read_chunks, k8, ks, ids, 0, block=32)
    no(shadowkv.kv8_read_chunks, k8, ks, ids.int(), 8, block=32)
    no(shadowkv.kv8_read_chunks, k8, ks, ids[:1], 8, block=32)
    no(shadowkv.kv8_read_chunks, k8, ks, ids.cpu(), 8, block=32)
    assert shadowkv.kv8_attn(q, *caches, at, block=32).abs().max() == 0  # (empty sequences, after all that)
