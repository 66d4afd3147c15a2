"""The operators of the 8-bit KV cache, as cases that can be timed and compared.

A cache of keys or values holds e4m3 codes [B, H, capacity, 128] and a scale (fp32, a power of two) for each
block of tokens and head [B, H, capacity / block]; a value is code * scale.

  write   new tokens' keys and values quantised into the cache where each sequence ends, the last block's
          scale raised (and its older rows encoded again) where a new row asks for it
  read    cached rows as bf16: a range of rows, or the chunks that a selection names
  attend  attention of new tokens, the last of their sequence, over the cached keys and values that they see:
          all up to their own, or a window of the last ones and a few first ones (sinks)

Sizes follow the model shapes of decode_model (32 query heads on 8 or 2 kv heads of 128 dims, contexts of 8192 to
262144 tokens, selections of 256 chunks of 8 rows). A case is a dict of plain values.
"""
import math

import torch

own = False

DEV = "cuda:0"
D = 128
E4M3 = torch.float8_e4m3fn


def listed():
    return [
        # One decoded token a sequence, batch 8 at different positions: latency.
        dict(name="write_token_b8", kind="write", batch=8, heads=8, rows=1, start=7001, ragged=True, block=64),
        # A chunk of a ragged batch of prompts, into blocks begun before.
        dict(name="write_ragged_b4", kind="write", batch=4, heads=2, rows=509, start=1021, ragged=True, block=32),
        # A whole prompt at the benchmark's context.
        dict(name="write_prompt_122k", kind="write", batch=1, heads=8, rows=122880, start=0, ragged=False, block=64),
        # The chunks of a sparse decode's selection, batch 8 at the benchmark's context.
        dict(name="read_chunks_b8", kind="read", batch=8, heads=8, rows=122880, chunks=256, chunk=8, block=64),
        # A sequence read back whole.
        dict(name="read_rows_100k", kind="read", batch=1, heads=8, rows=100003, chunks=0, chunk=1, block=128),
        # One token of one sequence of a thousand: latency.
        dict(name="token_b1_1k", kind="attend", batch=1, heads=8, group=4, rows=1, length=1000, ragged=False, window=0,
             sinks=0, block=64),
        # A decode step's layer at batch 8 and the benchmark's context.
        dict(name="token_b8_122k", kind="attend", batch=8, heads=8, group=4, rows=1, length=122880, ragged=False,
             window=0, sinks=0, block=64),
        # 2 kv heads of 16 query heads at 262144 tokens.
        dict(name="token_b4_262k_g16", kind="attend", batch=4, heads=2, group=16, rows=1, length=262143, ragged=False,
             window=0, sinks=0, block=128),
        # A serving batch of very different lengths under a sliding window with sinks.
        dict(name="token_b24_window", kind="attend", batch=24, heads=8, group=4, rows=1, length=61441, ragged=True,
             window=8192, sinks=64, block=64),
        # A few drafted tokens a sequence, to be verified.
        dict(name="draft_b4_30k", kind="attend", batch=4, heads=8, group=4, rows=5, length=30011, ragged=True, window=0,
             sinks=0, block=32),
        # A prompt of 8192 tokens.
        dict(name="prompt_8k", kind="attend", batch=1, heads=8, group=4, rows=8192, length=8192, ragged=False, window=0,
             sinks=0, block=64),
        # A later piece of two long prompts, under a window with sinks.
        dict(name="piece_2k_window", kind="attend", batch=2, heads=2, group=16, rows=2048, length=33333, ragged=True,
             window=8192, sinks=16, block=64),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    heads, group = rng.choice([(8, 4), (2, 16), (4, 1), (1, 7)])
    block = rng.choice([16, 32, 64, 128])
    kind = rng.choice(["write", "read", "token", "attend"])
    if kind == "write":
        batch = _log(rng, 1, 16)
        rows = _log(rng, 1, min(122880, 900000 // (batch * heads)))
        return dict(kind="write", batch=batch, heads=heads, rows=rows, start=rng.choice([0, _log(rng, 1, 16384)]),
                    ragged=rng.random() < 0.5, block=block)
    if kind == "read":
        batch = _log(rng, 1, 16)
        chunks = rng.choice([0, _log(rng, 1, 512)])
        rows = _log(rng, 600, min(122880, 2000000 // (batch * heads)))
        return dict(kind="read", batch=batch, heads=heads, rows=rows, chunks=chunks,
                    chunk=rng.choice([4, 8, 16]) if chunks else 1, block=block)
    window = rng.choice([0, _log(rng, 128, 16384)])
    sinks = rng.choice([0, 4, _log(rng, 1, 256)]) if window else 0
    batch = _log(rng, 1, 32 if kind == "token" else 8)
    length = _log(rng, 1 if kind == "token" else 64, min(262144, 7000000 // (batch * heads)))
    rows = 1
    if kind == "attend":
        rows = _log(rng, 2, max(2, min(length, 1600000000 // (batch * heads * group * length), 8192)))
    return dict(kind="attend", batch=batch, heads=heads, group=group, rows=rows, length=length,
                ragged=rng.random() < 0.5, window=window, sinks=sinks, block=block)


def _lengths(most, batch, ragged):
    """Tokens of each sequence: the longest `most`, the others spread below it where they are ragged."""
    return [max(1, most - (most * b) // batch - 3 * (b % 5)) if ragged else most for b in range(batch)]


def _counts(case):
    """New tokens of each sequence (of `rows` at most), for a write or an attention."""
    return [max(1, case["rows"] - (case["rows"] * b) // (2 * case["batch"])) if case["ragged"] else case["rows"]
            for b in range(case["batch"])]


def _starts(case):
    return [case["start"] + (13 * b if case["ragged"] else 0) for b in range(case["batch"])]


def _totals(case):
    """Tokens of each sequence of an attention, its new ones among them."""
    return [max(n, m) for n, m in zip(_counts(case), _lengths(case["length"], case["batch"], case["ragged"]))]


def _capacity(rows, block):
    return (rows // block + 2) * block


def _pow2_scale(amax):
    """The smallest power of two (2^-126 at least) under which amax is at most 448."""
    m, e = torch.frexp(amax)  # amax = m * 2^e, m in [0.5, 1)
    e = torch.where(amax > 0, e - 9 + (m > 0.875).to(e.dtype), torch.full_like(e, -126)).clamp(min=-126)
    return torch.ldexp(torch.ones_like(amax), e)


def _pack(x, block):
    """x [B, H, rows, 128] (rows a multiple of block) -> codes and scales, for the caches that prepare() fills."""
    B, H, n, _ = x.shape
    g = x.view(B, H, n // block, block * D)
    s = _pow2_scale(g.abs().amax(-1))
    return (g / s.unsqueeze(-1)).view(B, H, n, D).to(E4M3), s


def _keys(B, H, n, gen):
    """Keys after the rotary embedding: some channels larger than others."""
    chan = torch.exp(0.5 * torch.randn(1, H, 1, D, generator=gen, device=DEV))
    return torch.randn(B, H, n, D, generator=gen, device=DEV) * chan


def _values(B, H, n, gen):
    mean = 0.2 * torch.randn(1, H, 1, D, generator=gen, device=DEV)
    return torch.randn(B, H, n, D, generator=gen, device=DEV) * 0.6 + mean


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    B, H, block = case["batch"], case["heads"], case["block"]
    st = dict(case=case)
    if case["kind"] == "write":
        T = case["rows"]
        # views of the projection's output, as a model has them
        st["k"] = _keys(B, H, T, gen).to(torch.bfloat16).transpose(1, 2).contiguous().transpose(1, 2)
        st["v"] = _values(B, H, T, gen).to(torch.bfloat16).transpose(1, 2).contiguous().transpose(1, 2)
        st["start"], st["counts"] = _ints(_starts(case)), _ints(_counts(case)) if case["ragged"] else None
        cap = _capacity(max(_starts(case)) + T, block)
        before = (max(_starts(case)) + block - 1) // block * block
        for name, make in (("k", _keys), ("v", _values)):
            codes = torch.zeros(B, H, cap, D, dtype=E4M3, device=DEV)
            scale = torch.full((B, H, cap // block), 2.0 ** -126, device=DEV)
            if before:
                codes.view(torch.uint8)[:, :, :before], scale[:, :, :before // block] = \
                    [t.view(torch.uint8) if t.dtype == E4M3 else t for t in _pack(make(B, H, before, gen), block)]
            st[name + "8"], st[name + "_scale"] = codes, scale
        return st
    rows = case["rows"] if case["kind"] == "read" else max(_totals(case))
    cap = _capacity(rows, block)
    if case["kind"] == "read":
        st["x8"], st["scale"] = _pack(_values(B, H, cap, gen), block)
        if case["chunks"]:
            n = rows // case["chunk"]
            ids = torch.rand(B, H, n, generator=gen, device=DEV).argsort(dim=-1)[:, :, :case["chunks"]]
            st["chunk_ids"] = ids.contiguous()
        return st
    T, Hq = case["rows"], H * case["group"]
    k, v = _keys(B, H, cap, gen), _values(B, H, cap, gen)
    st["k8"], st["k_scale"] = _pack(k, block)
    st["v8"], st["v_scale"] = _pack(v, block)
    q = torch.randn(B, T, Hq, D, generator=gen, device=DEV) * 1.2
    st["q"] = q.to(torch.bfloat16).transpose(1, 2)
    st["lengths"], st["counts"] = _ints(_totals(case)), _ints(_counts(case)) if case["ragged"] else None
    return st


def _plain_write_one(x, codes, scale, start, counts, block):
    B, H, T, _ = x.shape
    cap = codes.shape[2]
    nb = (T + block - 2) // block + 1  # blocks that T rows can touch
    b = torch.arange(B, device=DEV).unsqueeze(1)
    blk = start.long().unsqueeze(1) // block + torch.arange(nb, device=DEV)
    pos = (blk.unsqueeze(2) * block + torch.arange(block, device=DEV)).view(B, -1)
    t = pos - start.unsqueeze(1)
    new = (t >= 0) & (t < counts.unsqueeze(1)) & (pos < cap)
    at = pos.clamp(max=cap - 1)
    rows = x.float().transpose(1, 2)[b, t.clamp(0, T - 1)]  # [B, nb * block, H, D]
    raw = codes.view(torch.uint8).transpose(1, 2)
    held = raw[b, at]
    was = scale.transpose(1, 2)[b, blk.clamp(max=scale.shape[2] - 1)]  # [B, nb, H]
    amax = torch.where(new.view(B, -1, 1, 1), rows, 0.0).abs().view(B, nb, block, H, D).amax((2, 4))
    need = _pow2_scale(amax)
    begun = (blk * block < start.unsqueeze(1)).unsqueeze(2)
    s = torch.where(begun, torch.maximum(was, need), need)
    touched = new.view(B, nb, block).any(2).unsqueeze(2)
    s = torch.where(touched, s, was)
    wide = lambda u: u.repeat_interleave(block, 1).unsqueeze(3)  # noqa: E731
    value = torch.where(new.view(B, -1, 1, 1), rows, held.view(E4M3).float() * wide(was))
    change = (new | (pos < start.unsqueeze(1))).view(B, -1, 1, 1) & wide(touched)
    raw[b, at] = torch.where(change, (value / wide(s)).to(E4M3).view(torch.uint8), held)
    scale.transpose(1, 2)[b, blk.clamp(max=scale.shape[2] - 1)] = s


def _plain_write(st):
    case = st["case"]
    counts = st["counts"] if st["counts"] is not None else torch.full_like(st["start"], case["rows"])
    _plain_write_one(st["k"], st["k8"], st["k_scale"], st["start"], counts, case["block"])
    _plain_write_one(st["v"], st["v8"], st["v_scale"], st["start"], counts, case["block"])


def _plain_values(codes, scale, block):
    return codes.float() * scale.repeat_interleave(block, 2)[:, :, :codes.shape[2]].unsqueeze(3)


def _plain_read(st):
    case = st["case"]
    B, H, block = case["batch"], case["heads"], case["block"]
    if not case["chunks"]:
        n = case["rows"]
        return _plain_values(st["x8"][:, :, :n], st["scale"], block).to(torch.bfloat16)
    c = case["chunk"]
    rows = (st["chunk_ids"].unsqueeze(3) * c + torch.arange(c, device=DEV)).view(B, H, -1)
    codes = st["x8"].view(torch.uint8).gather(2, rows.unsqueeze(3).expand(-1, -1, -1, D)).view(E4M3)
    return (codes.float() * st["scale"].gather(2, rows // block).unsqueeze(3)).to(torch.bfloat16)


def _plain_attend(st):
    case = st["case"]
    B, H, G, T, block = case["batch"], case["heads"], case["group"], case["rows"], case["block"]
    L = max(_totals(case))  # (of the case: nothing is asked of the GPU)
    counts = st["counts"] if st["counts"] is not None else torch.full_like(st["lengths"], T)
    k = _plain_values(st["k8"][:, :, :L], st["k_scale"], block)
    v = _plain_values(st["v8"][:, :, :L], st["v_scale"], block)
    q = st["q"].reshape(B, H, G * T, D).float()
    s = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(D))
    t, j = torch.arange(T, device=DEV).view(1, T, 1), torch.arange(L, device=DEV)
    p = (st["lengths"] - counts).view(B, 1, 1) + t
    see = (j <= p) & (t < counts.view(B, 1, 1))
    if case["window"]:
        see = see & ((j > p - case["window"]) | (j < case["sinks"]))
    s = s.view(B, H, G, T, L).masked_fill(~see.view(B, 1, 1, T, L), -math.inf)
    top = s.amax(-1, keepdim=True)
    w = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    del s
    out = torch.matmul(w.view(B, H, G * T, L), v) / w.sum(-1).clamp(min=1e-30).view(B, H, G * T, 1)
    return out.view(B, H * G, T, D).transpose(1, 2).to(torch.bfloat16)


def run(state):
    case = state["case"]
    kind, block = case["kind"], case["block"]
    if own:
        from shadowkv_amd.kernels import shadowkv
        if kind == "write":
            shadowkv.kv8_write(state["k"], state["v"], state["k8"], state["v8"], state["k_scale"], state["v_scale"],
                               state["start"], counts=state["counts"], block=block)
            return [state["k8"], state["v8"], state["k_scale"], state["v_scale"]]
        if kind == "read":
            if case["chunks"]:
                return shadowkv.kv8_read_chunks(state["x8"], state["scale"], state["chunk_ids"], case["chunk"],
                                                block=block)
            return shadowkv.kv8_read(state["x8"], state["scale"], 0, case["rows"], block=block)
        return shadowkv.kv8_attn(state["q"], state["k8"], state["v8"], state["k_scale"], state["v_scale"],
                                 state["lengths"], counts=state["counts"], block=block,
                                 window=case["window"] or None, sinks=case["sinks"])
    if kind == "write":
        _plain_write(state)
        return [state["k8"], state["v8"], state["k_scale"], state["v_scale"]]
    return _plain_read(state) if kind == "read" else _plain_attend(state)


def _pairs(n, total, window, sinks):
    """(query, key) pairs that the last n tokens of `total` see, and the keys that any of them sees."""
    pairs = 0
    if not window:
        pairs = n * total - n * (n - 1) // 2
        return pairs, total
    for p in range(total - n, total):
        lo = max(0, p - window + 1)
        pairs += p + 1 - lo + min(sinks, lo)
    lo = max(0, total - n - window + 1)
    return pairs, total - lo + min(sinks, lo)


def work(case):
    B, H, block = case["batch"], case["heads"], case["block"]
    if case["kind"] == "write":
        rows = sum(_counts(case))
        return dict(bytes=2 * H * (rows * 3 * D + 8 * (rows // block + B)), flops=0)
    if case["kind"] == "read":
        rows = B * (case["chunks"] * case["chunk"] or case["rows"])
        return dict(bytes=H * (rows * 3 * D + 4 * (rows // block + 1)), flops=0)
    pairs = keys = 0
    for n, total in zip(_counts(case), _totals(case)):
        p, k = _pairs(n, total, case["window"], case["sinks"])
        pairs, keys = pairs + p, keys + k
    Hq = H * case["group"]
    return dict(bytes=keys * H * (2 * D + 8 / block) + 4 * sum(_counts(case)) * Hq * D, flops=4 * D * Hq * pairs)


def _e4m3(x):
    """x (64 bits, at most 448 large) at the nearest e4m3 value, ties to the even one: 3 bits after the first, steps
    of 2^-9 at least."""
    step = torch.exp2(torch.frexp(x)[1].double() - 4).clamp(min=2.0 ** -9)
    return torch.round(x / step) * step


def _exact_write(case, st):
    block, out = case["block"], []
    for name in ("k", "v"):
        codes, scale = st[name + "8"].double(), st[name + "_scale"].double()
        for b, (a, n) in enumerate(zip(_starts(case), _counts(case))):
            first = a // block * block
            whole = -(-(a + n) // block) * block
            value = torch.zeros(case["heads"], whole - first, D, dtype=torch.float64, device=DEV)
            value[:, a - first:a - first + n] = st[name][b, :, :n].double()
            g = value.view(case["heads"], -1, block * D)
            amax = g.abs().amax(-1)
            need = torch.where(amax > 0, torch.exp2(torch.ceil(torch.log2(amax / 448)).clamp(min=-126)), 2.0 ** -126)
            old = scale[b, :, first // block].clone()
            if a > first:
                need[:, 0] = torch.maximum(need[:, 0], old)
                g[:, 0, :(a - first) * D] = (codes[b, :, first:a] * old.view(-1, 1, 1)).flatten(1)
            coded = _e4m3(g / need.unsqueeze(2)).view(case["heads"], -1, D)
            codes[b, :, first:a + n] = coded[:, :a + n - first]
            scale[b, :, first // block:whole // block] = need
        out += [codes, scale]
    return [out[0], out[2], out[1], out[3]]


def exact(case, seed):
    st = prepare(case, seed)
    B, H, block = case["batch"], case["heads"], case["block"]
    if case["kind"] == "write":
        return _exact_write(case, st)
    if case["kind"] == "read":
        n = case["rows"]
        out = torch.repeat_interleave(st["scale"].double(), block, dim=2)[..., None] * st["x8"].double()
        if not case["chunks"]:
            return out[:, :, :n]
        c = case["chunk"]
        whole = out[:, :, :n // c * c].unflatten(2, (n // c, c))
        return torch.stack([torch.stack([whole[b, h, st["chunk_ids"][b, h]].flatten(0, 1) for h in range(H)])
                            for b in range(B)])
    G, T = case["group"], case["rows"]
    out = torch.zeros(B, T, H * G, D, dtype=torch.float64, device=DEV)
    for b, (n, total) in enumerate(zip(_counts(case), _totals(case))):
        for h in range(H):
            k, v = [st[x + "8"][b, h, :total].double()
                    * st[x + "_scale"][b, h].double().repeat_interleave(block)[:total, None] for x in ("k", "v")]
            at = torch.arange(total - n, total, device=DEV)[:, None]
            key = torch.arange(total, device=DEV)[None]
            hidden = key > at
            if case["window"]:
                hidden |= (key <= at - case["window"]) & (key >= case["sinks"])
            for g in range(G):
                s = (st["q"][b, h * G + g, :n].double() @ k.T) / math.sqrt(D)
                out[b, :n, h * G + g] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ v
    return out
