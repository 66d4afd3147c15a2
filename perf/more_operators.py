"""The operators of a paged KV cache, as cases that can be timed and compared.

Keys and values lie in pages [pages, H, page, 128] (bf16) that sequences of different lengths share: a sequence's
table names its pages in order. A step brings some new tokens of each sequence, packed one behind the other.

  tables  a step's pages taken from the free ones, where its tokens begin in the packed rows and where each is to be
          stored, and then the same pages given back (a step whose tokens are all dropped)
  write   a step's keys and values into the pages
  prompt  causal attention of whole prompts, packed
  paged   attention of a step's queries, the last tokens of their sequences, over the pages: all keys up to their
          own, or a window of the last ones

Sizes follow the model shapes of decode_model (32 query heads on 8 or 2 kv heads of 128 dims, contexts up to 122880
tokens). A case is a dict of plain values.
"""
import math

import torch

own = False

DEV = "cuda:0"
D = 128
BF16 = torch.bfloat16


def listed():
    return [
        # A decode step of 64 sequences: latency.
        dict(name="tables_decode_b64", kind="tables", batch=64, rows=1, length=8000, ragged=True, page=64, pad=0),
        # Pieces of the prompts of 256 sequences in one step, small pages, in a step buffer larger than they are.
        dict(name="tables_pieces_b256", kind="tables", batch=256, rows=301, length=12000, ragged=True, page=16, pad=777),
        # One new token of each of 64 sequences: latency.
        dict(name="write_decode_b64", kind="write", batch=64, heads=8, rows=1, length=3000, ragged=True, page=64,
             order="head", pad=0),
        # A step of prompts into pages that hold a token's heads together, with room behind the last token.
        dict(name="write_prompts_b8", kind="write", batch=8, heads=8, rows=4099, length=6000, ragged=True, page=16,
             order="token", pad=333),
        # Three short prompts: latency.
        dict(name="prompt_short_b3", kind="prompt", batch=3, heads=8, group=4, rows=131, ragged=True, window=0, pad=0),
        # A batch of prompts of very different lengths, up to 4096.
        dict(name="prompt_ragged_b8", kind="prompt", batch=8, heads=8, group=4, rows=4096, ragged=True, window=0, pad=64),
        # Two long prompts, 16 query heads on each of 2 kv heads.
        dict(name="prompt_long_b2_g16", kind="prompt", batch=2, heads=2, group=16, rows=16001, ragged=True, window=0,
             pad=0),
        # One token of one sequence of a thousand: latency.
        dict(name="token_b1_1k", kind="paged", batch=1, heads=8, group=4, rows=1, singles=1, length=1000, ragged=False,
             window=0, page=64, order="head", pad=0),
        # A decode step's layer of 16 sequences of up to 122880 tokens.
        dict(name="token_b16_122k", kind="paged", batch=16, heads=8, group=4, rows=1, singles=16, length=122880,
             ragged=True, window=0, page=64, order="head", pad=0),
        # A few drafted tokens of each of 6 sequences, to be verified, small pages that hold a token's heads together.
        dict(name="draft_b6_30k", kind="paged", batch=6, heads=8, group=4, rows=5, singles=0, length=30011, ragged=True,
             window=0, page=16, order="token", pad=0),
        # A serving step: a piece of one long prompt beside one token of each of 23 other sequences, under a window.
        dict(name="mixed_b24_window", kind="paged", batch=24, heads=2, group=16, rows=1024, singles=23, length=61441,
             ragged=True, window=8192, page=128, order="head", pad=17),
        # A later piece of two long prompts.
        dict(name="piece_2k_b2_60k", kind="paged", batch=2, heads=8, group=4, rows=2048, singles=0, length=60003,
             ragged=True, window=0, page=64, order="head", pad=0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    heads, group = rng.choice([(8, 4), (2, 16), (4, 1), (1, 7)])
    page = rng.choice([16, 32, 64, 128, 256])
    pad = rng.choice([0, 0, _log(rng, 1, 300)])
    kind = rng.choice(["tables", "write", "prompt", "prompt", "paged", "paged", "paged"])
    if kind == "tables":
        batch = _log(rng, 1, 256)
        rows = _log(rng, 1, min(16384, 70000 // batch))
        return dict(kind="tables", batch=batch, rows=rows, length=_log(rng, rows, 32768), ragged=rng.random() < 0.7,
                    page=page, pad=pad)
    if kind == "write":
        batch = _log(rng, 1, 64)
        rows = _log(rng, 1, min(16384, 200000 // (batch * heads)))
        return dict(kind="write", batch=batch, heads=heads, rows=rows, length=rows + _log(rng, 1, 2000),
                    ragged=rng.random() < 0.7, page=page, order=rng.choice(["head", "token"]), pad=pad)
    window = rng.choice([0, 0, _log(rng, 64, 16384)])
    if kind == "prompt":
        batch = _log(rng, 1, 16)
        most = math.isqrt(2 * 4000000000 // (batch * heads * group))
        return dict(kind="prompt", batch=batch, heads=heads, group=group, rows=_log(rng, 1, min(16384, most)),
                    ragged=rng.random() < 0.7, window=window, pad=pad)
    batch = _log(rng, 1, 32)
    length = _log(rng, 16, min(122880, 7000000 // (batch * heads)))
    form = rng.choice(["token", "draft", "piece", "mixed"])
    rows = 1
    if form == "draft":
        rows = min(length, rng.randint(2, 8))
    elif form != "token":
        rows = _log(rng, 2, max(2, min(length, 4000000000 // (batch * heads * group * length), 8192)))
    singles = batch if form == "token" else batch - 1 if form == "mixed" else 0
    return dict(kind="paged", batch=batch, heads=heads, group=group, rows=rows, singles=singles, length=length,
                ragged=rng.random() < 0.7, window=window, page=page, order=rng.choice(["head", "token"]), pad=pad)


def _counts(case):
    """New tokens of each sequence: of `rows` at most, one of the last `singles`."""
    B, n, single = case["batch"], case["rows"], case.get("singles", 0)
    return [1 if b >= B - single else max(1, n - (n * 3 * b) // (4 * B) - b % 3) if case["ragged"] else n
            for b in range(B)]


def _totals(case):
    """Tokens of each sequence, its new ones among them."""
    n = _counts(case)
    if case["kind"] == "prompt":
        return n
    B, most = case["batch"], case["length"]
    return [max(c, most - (most * b) // B - 3 * (b % 5)) if case["ragged"] else max(c, most) for b, c in enumerate(n)]


def _begins(case):
    out = [0]
    for n in _counts(case):
        out.append(out[-1] + n)
    return out


def _rows(case):
    return _begins(case)[-1] + case["pad"]


def _need(tokens, page):
    return -(-tokens // page)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _qkv(n, heads, gen, std, spread):
    """A projection's output, of which q, k and v are views: [n, sum(heads), 128], some channels larger than others
    where spread is not zero, some with a mean."""
    parts = []
    for h, s, e in zip(heads, std, spread):
        x = torch.randn(n, h, D, generator=gen, device=DEV) * s
        if e:
            x = x * torch.exp(e * torch.randn(1, h, D, generator=gen, device=DEV))
        else:
            x = x + 0.2 * torch.randn(1, h, D, generator=gen, device=DEV)
        parts.append(x.to(BF16))
    return torch.cat(parts, 1).split(list(heads), 1)


def _pages(pages, heads, page, order, gen, spread):
    """A layer's pages, keys (spread) or values, as [pages, heads, page, 128]."""
    shape = (pages, heads, page, D) if order == "head" else (pages, page, heads, D)
    out = torch.empty(shape, dtype=BF16, device=DEV)
    per_head = (1, heads, 1, D) if order == "head" else (1, 1, heads, D)
    chan = torch.randn(per_head, generator=gen, device=DEV)
    step = max(1, (1 << 28) // (heads * page * D))
    for i in range(0, pages, step):
        x = torch.randn(min(step, pages - i), *shape[1:], generator=gen, device=DEV)
        out[i:i + step] = x * torch.exp(0.5 * chan) if spread else 0.6 * x + 0.2 * chan
    return out if order == "head" else out.transpose(1, 2)


def _table(case, totals, gen, width):
    """The pages of sequences of `totals` tokens, in no order: their tables, how many each holds, the free pages."""
    page, held = case["page"], [_need(n, case["page"]) for n in totals]
    spare = sum(_need(n, page) + 1 for n in _counts(case)) + 7
    ids = torch.randperm(sum(held) + spare, generator=gen, device=DEV).to(torch.int32)
    table = torch.full((case["batch"], width), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = ids[at:at + n]
        at += n
    return table, held, ids[at:].clone(), at + spare


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    st = dict(case=case, cu=_ints(_begins(case)))
    n, totals, counts = _rows(case), _totals(case), _counts(case)
    if case["kind"] == "prompt":
        H, G = case["heads"], case["group"]
        st["q"], st["k"], st["v"] = _qkv(n, (H * G, H, H), gen, (1.2, 1.0, 0.6), (0, 0.5, 0))
        return st
    page = case["page"]
    width = _need(max(totals), page) + 3
    if case["kind"] == "tables":
        before = [t - c for t, c in zip(totals, counts)]
        st["table"], held, free, _ = _table(case, before, gen, width)
        st["free_pages"] = torch.cat([free, torch.full((sum(held),), -1, dtype=torch.int32, device=DEV)])
        st["free_count"], st["held"] = _ints([free.numel()]), _ints(held)
        st["lengths"], st["counts"] = _ints(before), _ints(counts)
        return st
    H, order = case["heads"], case["order"]
    st["table"], _, _, pages = _table(case, totals, gen, width)
    st["k_pages"] = _pages(pages, H, page, order, gen, True)
    st["v_pages"] = _pages(pages, H, page, order, gen, False)
    if case["kind"] == "write":
        _, st["k"], st["v"] = _qkv(n, (4 * H, H, H), gen, (1.2, 1.0, 0.6), (0, 0.5, 0))
        slots = torch.full((n,), -1, dtype=torch.int32, device=DEV)
        for b, (a, c) in enumerate(zip(_begins(case), counts)):
            at = torch.arange(totals[b] - c, totals[b], device=DEV)
            slots[a:a + c] = st["table"][b][at // page] * page + (at % page).to(torch.int32)
        st["slots"] = slots
        return st
    st["lengths"] = _ints(totals)
    st["q"] = _qkv(n, (H * case["group"],), gen, (1.2,), (0,))[0]
    return st


# The plain forms.

def _plain_tables(st):
    case = st["case"]
    page, B, rows = case["page"], case["batch"], _rows(st["case"])
    table, held, free, count = st["table"], st["held"], st["free_pages"], st["free_count"]
    width = table.shape[1]
    lengths, counts = st["lengths"].long(), st["counts"].long().clamp(min=0)
    ends = counts.cumsum(0)
    total = lengths + counts
    ok = (total <= width * page) & ((ends <= rows) | (counts == 0))
    need = ((total + page - 1) // page - held).clamp(min=0) * (ok & (counts > 0))
    upto = need.cumsum(0)
    ok &= (need == 0) | (upto <= count)
    need = need * ok
    begin = upto - need
    totals = torch.where(ok, total, 0)
    cu = torch.cat([torch.zeros_like(ends[:1]), ends]).clamp(max=rows)
    p = torch.arange(width, device=DEV)
    i = p - held.long().unsqueeze(1)
    new = (i >= 0) & (i < need.unsqueeze(1))
    table.copy_(torch.where(new, free[(count - 1 - begin.unsqueeze(1) - i).clamp(0, free.numel() - 1)], table))
    held.add_(need)
    count.sub_(need.sum())
    r = torch.arange(rows, device=DEV)
    b = torch.searchsorted(ends, r, right=True)
    inside = b < B
    b = b.clamp(max=B - 1)
    at = (lengths[b] + r - cu[b]).clamp(0, width * page - 1)
    slots = torch.where(inside & ok[b], table[b, at // page].long() * page + at % page, -1)
    # and back: what the tokens held before need stays
    stay = (lengths + page - 1) // page
    out = (held - stay).clamp(min=0)
    begin = out.cumsum(0) - out
    total_out = out.sum()
    i = p - stay.unsqueeze(1)
    old = (i >= 0) & (i < out.unsqueeze(1))
    to = torch.where(old, count + total_out - 1 - begin.unsqueeze(1) - i, free.numel())
    grown = torch.cat([free, free[:1]])
    grown.scatter_(0, to.flatten(), table.flatten())
    free.copy_(grown[:-1])
    table.masked_fill_(old, -1)
    held.sub_(out)
    count.add_(total_out)
    return [cu.to(torch.int32), totals.to(torch.int32), slots.to(torch.int32)]


def _plain_write(st):
    page = st["case"]["page"]
    slots = st["slots"][:_begins(st["case"])[-1]].long()  # (the others are -1)
    for x, pages in ((st["k"], st["k_pages"]), (st["v"], st["v_pages"])):
        pages[slots // page, :, slots % page] = x[:slots.numel()]


def _plain_softmax(q, k, v, n, window):
    """q [Hq, n, 128], the last n positions of k, v [H, L, 128] -> [n, Hq, 128]."""
    H, L, _ = k.shape
    at = torch.arange(L - n, L, device=DEV).unsqueeze(1)
    key = torch.arange(L, device=DEV)
    hidden = key > at
    if window:
        hidden = hidden | (key <= at - window)
    G = q.shape[0] // H
    out = torch.empty(n, H * G, D, dtype=BF16, device=DEV)
    each = max(1, min(G, (1 << 30) // (n * L)))  # query heads at a time
    for h in range(H):
        for g in range(0, G, each):
            x = q[h * G + g:h * G + min(g + each, G)]
            s = torch.matmul(x.reshape(-1, D), k[h].t()).view(-1, n, L) * (1.0 / math.sqrt(D))
            s.masked_fill_(hidden, -math.inf)
            s.sub_(s.amax(-1, keepdim=True)).exp_()
            o = torch.matmul(s.view(-1, L), v[h]).view(-1, n, D) / s.sum(-1, keepdim=True)
            out[:, h * G + g:h * G + g + o.shape[0]] = o.transpose(0, 1)
    return out


def _plain_attention(st):
    case = st["case"]
    begins, totals, window = _begins(case), _totals(case), case["window"]
    out = torch.zeros(_rows(case), st["q"].shape[1], D, dtype=BF16, device=DEV)
    for b in range(case["batch"]):
        rows = slice(begins[b], begins[b + 1])
        if case["kind"] == "prompt":
            k, v = (st[x][rows].float().transpose(0, 1).contiguous() for x in "kv")
        else:
            ids = st["table"][b, :_need(totals[b], case["page"])].long()
            k, v = (st[x][ids].float().transpose(0, 1).reshape(case["heads"], -1, D)[:, :totals[b]]
                    for x in ("k_pages", "v_pages"))
        out[rows] = _plain_softmax(st["q"][rows].float().transpose(0, 1), k, v, begins[b + 1] - begins[b], window)
    return out


def _own(st):
    from shadowkv_amd.kernels import shadowkv
    case = st["case"]
    if case["kind"] == "tables":
        step = shadowkv.paged_reserve(st["lengths"], st["counts"], st["table"], st["held"], st["free_pages"],
                                      st["free_count"], rows=_rows(case), page=case["page"])
        shadowkv.paged_release(st["lengths"], st["lengths"], st["table"], st["held"], st["free_pages"],
                               st["free_count"], page=case["page"])
        return list(step)
    if case["kind"] == "write":
        return shadowkv.paged_write(st["k"], st["v"], st["k_pages"], st["v_pages"], st["slots"])
    window = case["window"] or None
    if case["kind"] == "prompt":
        return shadowkv.packed_attn(st["q"], st["k"], st["v"], st["cu"], window=window)
    return shadowkv.paged_attn(st["q"], st["k_pages"], st["v_pages"], st["table"], st["lengths"], st["cu"],
                               max_new=case["rows"], window=window)


def run(state):
    kind = state["case"]["kind"]
    if own:
        out = _own(state)
    else:
        out = (_plain_tables if kind == "tables" else _plain_write if kind == "write" else _plain_attention)(state)
    if kind == "tables":
        return out + [state[x] for x in ("table", "held", "free_pages", "free_count", "lengths")]
    return [state["k_pages"], state["v_pages"]] if kind == "write" else out


def _pairs(n, total, window):
    """(query, key) pairs that the last n tokens of `total` see, and the keys that any of them sees."""
    if not window:
        return n * total - n * (n - 1) // 2, total
    full = max(0, min(n, total - window + 1))  # queries whose window is whole
    first = n - full  # those at positions total - n ...
    return full * window + first * (total - n + 1) + first * (first - 1) // 2, min(total, n + window - 1)


def work(case):
    rows, B = _begins(case)[-1], case["batch"]
    if case["kind"] == "tables":
        page = case["page"]
        new = sum(_need(t, page) - _need(t - c, page) for t, c in zip(_totals(case), _counts(case)))
        entries = sum(_need(t, page) - (t - c) // page for t, c in zip(_totals(case), _counts(case)))
        return dict(bytes=4 * (_rows(case) + entries + 6 * new + 8 * B), flops=0)
    H = case["heads"]
    if case["kind"] == "write":
        return dict(bytes=rows * (8 * H * D + 4), flops=0)
    pairs = keys = 0
    for n, total in zip(_counts(case), _totals(case)):
        p, k = _pairs(n, total, case["window"])
        pairs, keys = pairs + p, keys + k
    Hq = H * case["group"]
    return dict(bytes=4 * keys * H * D + 4 * _rows(case) * Hq * D, flops=4 * D * Hq * pairs)


# The definitions, one step after the other.

def _exact_tables(case, st):
    page, rows = case["page"], _rows(case)
    table, held, free = (st[x].tolist() for x in ("table", "held", "free_pages"))
    lengths, counts, left = st["lengths"].tolist(), st["counts"].tolist(), st["free_count"].item()
    cu, totals, slots = [0], [], [-1] * rows
    asked, top = 0, left
    for b, (have, new) in enumerate(zip(lengths, counts)):
        cu.append(min(cu[-1] + new, rows))
        served = have + new <= len(table[b]) * page and cu[-1] - cu[-2] == new
        more = max(0, -(-(have + new) // page) - held[b]) if served and new else 0
        asked += more
        if more and asked > top:
            served = False
        totals.append(have + new if served else 0)
        if not served:
            continue
        for _ in range(more):
            left -= 1
            table[b][held[b]] = free[left]
            held[b] += 1
        for t in range(new):
            slots[cu[-2] + t] = table[b][(have + t) // page] * page + (have + t) % page
    for b in reversed(range(len(held))):
        while held[b] > -(-lengths[b] // page):
            held[b] -= 1
            free[left] = table[b][held[b]]
            table[b][held[b]] = -1
            left += 1
    return [torch.tensor(x, dtype=torch.int64) for x in (cu, totals, slots, table, held, free, [left], lengths)]


def _exact_attention(case, st):
    H, G, window = case["heads"], case["group"], case["window"]
    out = torch.zeros(_rows(case), H * G, D, dtype=torch.float64, device=DEV)
    begins = _begins(case)
    for b, total in enumerate(_totals(case)):
        first, n = begins[b], begins[b + 1] - begins[b]
        i = torch.arange(n, device=DEV).view(n, 1) + total - n
        j = torch.arange(total, device=DEV).view(1, total)
        seen = j <= i
        if window:
            seen &= i - j < window
        if case["kind"] == "paged":
            where = st["table"][b].long()[j[0] // case["page"]], j[0] % case["page"]
        for h in range(H):
            if case["kind"] == "prompt":
                k, v = st["k"][first:first + n, h].double(), st["v"][first:first + n, h].double()
            else:
                k, v = st["k_pages"][:, h][where].double(), st["v_pages"][:, h][where].double()
            for g in range(h * G, h * G + G):
                s = st["q"][first:first + n, g].double() @ k.T / D ** 0.5
                out[first:first + n, g] = torch.where(seen, s, -math.inf).softmax(1) @ v
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "tables":
        return _exact_tables(case, st)
    if case["kind"] != "write":
        return _exact_attention(case, st)
    out = []
    slots = st["slots"].tolist()
    for x, pages in ((st["k"], st["k_pages"]), (st["v"], st["v_pages"])):
        want = pages.double().permute(0, 2, 1, 3).reshape(-1, *x.shape[1:])
        rows = [r for r, s in enumerate(slots) if s >= 0]
        want.index_copy_(0, torch.tensor([slots[r] for r in rows], device=DEV), x.double()[rows])
        out.append(want.view(-1, case["page"], *x.shape[1:]).permute(0, 2, 1, 3))
    return out
