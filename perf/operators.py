"""Cases of the serving operators around a paged key-value cache: what is measured and the plain form of each.

  rotary      rotate the queries and keys of a batch of tokens and write keys and values to their pages
  attention   attention of one new token per sequence over its pages
  pages       fork sequences (share full pages, copy the last partial one), give them room for a token; compact a pool
  beam        choose the next beams over all continuations and reorder the beams' token histories

Where ``own`` is false, ``run`` computes them with elementary torch operations; where it is true it calls the framework.
A page pool is one tensor [planes, pages, ...page]; a sequence's table lists its pages in order; a page holds
``page`` consecutive positions of every kv head.  order "row": [pages, page, heads, dim] in memory, "head":
[pages, heads, page, dim], seen through a permuted view.
"""
import functools
import math

import numpy as np
import torch

own = False


@functools.lru_cache(None)
def _device():
    from tensorlib_amd import HipDevice
    return HipDevice(torch.cuda.current_device())


# ------------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # One token of one sequence, 32 heads of 128 and interleaved pairs as the Llama2-7B driver has them: latency.
        dict(name="rotary-1-token", op="rotary", seqs=1, tokens=1, start=1000, heads=32, kv_heads=32, dim=128, rotary=128,
             layout="interleaved", scaling="none", page=16, order="row"),
        # One decode step of a batch of 96 sequences, 3/4 of the head left unrotated, 80 wide heads.
        dict(name="rotary-decode-96", op="rotary", seqs=96, tokens=96, start=7000, heads=32, kv_heads=8, dim=80, rotary=20,
             layout="half", scaling="linear", page=32, order="head"),
        # Ragged prompts of a batch written at once, far positions with frequencies scaled for a long context.
        dict(name="rotary-prompts", op="rotary", seqs=7, tokens=16001, start=100000, heads=32, kv_heads=8, dim=128, rotary=128,
             layout="half", scaling="parts", page=16, order="row"),
        # A single sequence at the Llama2-7B context: the batch-1 decode step.
        dict(name="attention-1x2048", op="attention", seqs=1, low=2048, high=2048, heads=32, kv_heads=32, dim=128, page=16, order="row"),
        # The shortest: a few sequences just begun, all heads on one kv head, odd lengths inside one page or two.
        dict(name="attention-short", op="attention", seqs=3, low=1, high=19, heads=8, kv_heads=1, dim=64, page=16, order="row"),
        # An ordinary serving batch: ragged lengths, grouped heads.
        dict(name="attention-ragged-64", op="attention", seqs=64, low=65, high=4097, heads=32, kv_heads=8, dim=128, page=16, order="row"),
        # Few sequences with a long context: the split over the length carries it.
        dict(name="attention-long-4", op="attention", seqs=4, low=100001, high=131072, heads=64, kv_heads=8, dim=128, page=64, order="head"),
        # One beam search step of one request: 4 beams, all layers of a small model.
        dict(name="fork-4", op="fork", requests=1, beams=4, dropped=2, length=200, table=128, page=16, planes=32, kv_heads=8, dim=64),
        # The step for 48 requests at once, with the 64 planes of 32 layers.
        dict(name="fork-48x4", op="fork", requests=48, beams=4, dropped=1, length=300, table=128, page=16, planes=64, kv_heads=4, dim=64),
        # A fragmented pool packed to its low end.
        dict(name="compact-4096", op="compact", seqs=100, live=2000, pages=4096, table=64, page=16, planes=16, kv_heads=8, dim=128),
        # Beam selection of one request over the vocabulary of the Llama2 driver.
        dict(name="beam-1x4", op="beam", batch=1, beams=4, vocab=32000, history=256),
        # Many requests, a larger odd vocabulary (rows start at odd addresses).
        dict(name="beam-24x8", op="beam", batch=24, beams=8, vocab=100003, history=1024),
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    op = rng.choice(["rotary", "attention", "attention", "fork", "compact", "beam"])
    if op == "rotary":
        tokens = _log(rng, 1, 16000)
        dim = rng.choice([64, 80, 96, 128, 256])
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 4])
        return dict(op=op, seqs=_log(rng, 1, min(tokens, 200)), tokens=tokens, start=_log(rng, 1, 200000), heads=heads, kv_heads=kv, dim=dim,
                    rotary=rng.choice([dim, dim // 2, dim // 4]), layout=rng.choice(["half", "interleaved"]),
                    scaling=rng.choice(["none", "linear", "base", "parts"]), page=rng.choice([8, 16, 24, 64]), order=rng.choice(["row", "head"]))
    if op == "attention":
        kv = rng.choice([1, 2, 4, 8, 16])
        dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
        # the number of cached positions stays below that of the longest listed case of these widths
        high = _log(rng, 1, 131072)
        most = max(1, min(128, (1 << 28) // (high * kv * dim)))
        seqs = _log(rng, 1, most)
        return dict(op=op, seqs=seqs, low=max(1, high // rng.choice([1, 2, 50])), high=high, heads=kv * rng.choice([1, 2, 3, 4, 8]), kv_heads=kv,
                    dim=dim, page=rng.choice([1, 8, 16, 20, 32, 64, 128]), order=rng.choice(["row", "head"]))
    if op == "fork":
        beams = rng.choice([2, 3, 4, 5, 8])
        page = rng.choice([8, 16, 32])
        return dict(op=op, requests=_log(rng, 1, 160 // beams), beams=beams, dropped=rng.randrange(0, beams), length=_log(rng, 20, 400), table=512 // page + 8,
                    page=page, planes=rng.choice([2, 16, 32, 64]), kv_heads=rng.choice([1, 2, 4]), dim=64)
    if op == "compact":
        live = _log(rng, 50, 2000)
        return dict(op=op, seqs=_log(rng, 1, 40), live=live, pages=_log(rng, live + 10, 4096), table=live, page=rng.choice([8, 16]),
                    planes=rng.choice([2, 8, 16]), kv_heads=rng.choice([1, 4, 8]), dim=rng.choice([64, 128]))
    return dict(op=op, batch=_log(rng, 1, 24), beams=rng.randrange(1, 9), vocab=_log(rng, 500, 100003), history=_log(rng, 32, 1024))


# ------------------------------------------------------------------------------------------------ inputs

def _lengths(n, low, high):
    """n lengths spread over [low, high], both ends among them: the same for every seed, so that the work is too."""
    f = (np.arange(n) * 0.6180339887498949) % 1.0
    x = np.floor(low + f * (high - low + 1)).astype(np.int64).clip(low, high)
    x[0] = high
    if n > 1:
        x[1] = low
    return x


def _pages_of(lengths, page):
    return (lengths + page - 1) // page


def _frequencies(c):
    """Radians per position of each rotated pair, in 64 bits; a plan that a program computes once for a model."""
    rd, base, factor, context = c["rotary"], 10000.0, 8.0, 4096.0
    i = torch.arange(rd // 2, dtype=torch.float64)
    if c["scaling"] == "base" and rd > 2:
        base = base * factor ** (rd / (rd - 2))
    f = base ** (-2.0 * i / rd)
    if c["scaling"] == "linear":
        f = f / factor
    if c["scaling"] == "parts":
        turns = context * f / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
    return f.to("cuda")


def _tables(pages_per_seq, n_pages, width, rng):
    """Disjoint pages for every sequence, drawn from the whole pool in no order; -1 behind a sequence's last page."""
    order = rng.permutation(n_pages).astype(np.int32)
    at = np.concatenate([[0], np.cumsum(pages_per_seq)])
    col = np.arange(width)[None, :]
    idx = np.minimum(at[:-1, None] + col, n_pages - 1)
    return np.where(col < pages_per_seq[:, None], order[idx], -1).astype(np.int32)


def _pool(shape, g, std=1.0):
    x = torch.empty(shape, dtype=torch.float16, device="cuda")
    return x.normal_(0.0, std, generator=g)


def _view(pool, order):
    return pool if order == "row" else pool.permute(0, 2, 1, 3)


def prepare(case, seed):
    c = case
    rng = np.random.RandomState(seed % (1 << 31))
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dev = lambda a, t=torch.int32: torch.from_numpy(np.ascontiguousarray(a)).to("cuda", t)  # noqa: E731
    s = dict(case=c)
    if c["op"] == "rotary":
        n, page = c["tokens"], c["page"]
        base = np.full(c["seqs"], n // c["seqs"])
        base[: n - base.sum()] += 1
        if c["seqs"] > 1:                                      # ragged: shift tokens between neighbours
            cut = int(base[0]) // 2
            base[0] -= cut
            base[-1] += cut
        first = c["start"] + np.arange(c["seqs"]) * 7 % 50     # every sequence goes on from a context of its own
        end = first + base
        # the prompt's own pages lie at the end of a table; the pages before belong to the context and are not touched
        lead = first // page
        own_pages = _pages_of(end, page) - lead
        width = int(_pages_of(end, page).max())
        n_pages = int(own_pages.sum()) + 8
        packed = _tables(own_pages, n_pages, int(own_pages.max()), rng)
        tables = np.full((c["seqs"], width), -1, np.int32)
        seq_ids = np.repeat(np.arange(c["seqs"]), base)
        for i in range(c["seqs"]):
            tables[i, lead[i]: lead[i] + own_pages[i]] = packed[i, : own_pages[i]]
        positions = np.concatenate([np.arange(a, b) for a, b in zip(first, end)])
        width_qkv = (c["heads"] + 2 * c["kv_heads"]) * c["dim"]
        qkv = _pool((n, width_qkv), g)                          # rows of one fused projection
        q, k, v = qkv.split([c["heads"] * c["dim"], c["kv_heads"] * c["dim"], c["kv_heads"] * c["dim"]], dim=1)
        s["q"], s["k"], s["v"] = (t.unflatten(1, (-1, c["dim"])) for t in (q, k, v))
        shape = (n_pages, page, c["kv_heads"], c["dim"]) if c["order"] == "row" else (n_pages, c["kv_heads"], page, c["dim"])
        s["k_pages"], s["v_pages"] = _view(_pool(shape, g), c["order"]), _view(_pool(shape, g), c["order"])
        s["positions"], s["seq_ids"], s["tables"], s["freq"] = dev(positions), dev(seq_ids), dev(tables), _frequencies(c)
        s["magnitude"] = 0.1 * math.log(8.0) + 1.0 if c["scaling"] == "parts" else 1.0
    elif c["op"] == "attention":
        lens = rng.permutation(_lengths(c["seqs"], c["low"], c["high"]))
        used = _pages_of(lens, c["page"])
        width = int(_pages_of(np.array([c["high"]]), c["page"])[0])
        n_pages = int(used.sum()) + 3
        s["tables"], s["lens"] = dev(_tables(used, n_pages, width, rng)), dev(lens)
        shape = (n_pages, c["page"], c["kv_heads"], c["dim"]) if c["order"] == "row" else (n_pages, c["kv_heads"], c["page"], c["dim"])
        s["k_pages"], s["v_pages"] = _view(_pool(shape, g), c["order"]), _view(_pool(shape, g), c["order"])
        s["q"] = _pool((c["seqs"], c["heads"], c["dim"]), g)
        s["scale"] = 1.0 / math.sqrt(c["dim"])
    elif c["op"] == "fork":
        rows, page = c["requests"] * c["beams"], c["page"]
        # beams of a request share the pages of its prompt (2/3 of the length) and have the rest of their own
        length = _lengths(c["requests"], max(2, c["length"] // 2), c["length"])
        shared = np.repeat((2 * length // 3) // page, c["beams"])
        lens = np.repeat(length, c["beams"])
        used = _pages_of(lens, page)
        n_pages = int((used - shared).sum() + shared[:: c["beams"]].sum()) + 2 * rows
        order = rng.permutation(n_pages).astype(np.int32)
        tables = np.full((rows, c["table"]), -1, np.int32)
        at = 0
        for r in range(rows):
            if r % c["beams"] == 0:
                prompt = order[at: at + shared[r]]
                at += shared[r]
            tables[r, : shared[r]] = prompt
            tables[r, shared[r]: used[r]] = order[at: at + used[r] - shared[r]]
            at += used[r] - shared[r]
        refs = np.bincount(tables[tables >= 0], minlength=n_pages)
        parents = np.empty(rows, np.int64)
        for i in range(c["requests"]):                          # `dropped` beams of each request give way to copies of others
            kept = rng.permutation(c["beams"])[: c["beams"] - c["dropped"]]
            p = np.concatenate([kept, rng.choice(kept, c["dropped"])])
            parents[i * c["beams"]: (i + 1) * c["beams"]] = i * c["beams"] + rng.permutation(p)
        s["tables"], s["lens"], s["refs"], s["parents"] = dev(tables), dev(lens), dev(refs), dev(parents)
        s["add"] = torch.ones(rows, dtype=torch.int32, device="cuda")
        s["pool"] = _pool((c["planes"], n_pages, page, c["kv_heads"], c["dim"]), g)
    elif c["op"] == "compact":
        used = np.full(c["seqs"], c["live"] // c["seqs"])
        used[: c["live"] - used.sum()] += 1
        tables = _tables(used, c["pages"], c["table"], rng)
        if c["seqs"] > 1:
            tables[1, 0] = tables[0, 0]                         # a shared page
        s["tables"], s["refs"] = dev(tables), dev(np.bincount(tables[tables >= 0], minlength=c["pages"]))
        s["pool"] = _pool((c["planes"], c["pages"], c["page"], c["kv_heads"], c["dim"]), g)
    else:
        rows = c["batch"] * c["beams"]
        s["logits"] = _pool((rows, c["vocab"]), g, 2.5)
        s["scores"] = -20.0 * torch.rand(rows, generator=g, device="cuda")
        s["finished"] = dev(rng.rand(rows) < 0.1, torch.bool)
        s["history"] = dev(rng.randint(0, c["vocab"], (rows, c["history"])))
        s["lens"] = dev(rng.randint(1, c["history"], rows))
        s["end"] = 2
    return s


# ------------------------------------------------------------------------------------------------ plain forms

def _rotate(x, positions, freq, layout, magnitude):
    rd = 2 * freq.numel()
    angle = positions.double()[:, None] * freq[None, :]
    cos, sin = (angle.cos() * magnitude).float()[:, None, :], (angle.sin() * magnitude).float()[:, None, :]
    x = x.float()
    r, rest = x[..., :rd], x[..., rd:]
    if layout == "half":
        a, b = r[..., : rd // 2], r[..., rd // 2:]
        r = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([r, rest], -1).half()


def _plain_rotary(s):
    c = s["case"]
    q = _rotate(s["q"], s["positions"], s["freq"], c["layout"], s["magnitude"])
    k = _rotate(s["k"], s["positions"], s["freq"], c["layout"], s["magnitude"])
    pos = s["positions"].long()
    pages = s["tables"][s["seq_ids"].long(), pos // c["page"]].long()
    s["k_pages"][pages, pos % c["page"]] = k
    s["v_pages"][pages, pos % c["page"]] = s["v"]
    return q, s["k_pages"], s["v_pages"]


def _plain_attention(s):
    c = s["case"]
    t = torch.arange(c["high"], device="cuda")
    valid = t[None, :] < s["lens"][:, None]
    pages = s["tables"].long()[:, t // c["page"]].clamp_min(0)
    k = s["k_pages"][pages, t % c["page"]].float()                        # [seqs, positions, kv heads, dim]
    v = torch.where(valid[:, :, None, None], s["v_pages"][pages, t % c["page"]].float(), 0.0)
    q = s["q"].float().unflatten(1, (c["kv_heads"], -1))                  # [seqs, kv heads, group, dim]
    score = torch.matmul(q, k.permute(0, 2, 3, 1)) * s["scale"]
    score = torch.where(valid[:, None, None, :], score, float("-inf"))
    p = torch.exp(score - score.amax(-1, keepdim=True))
    out = torch.matmul(p, v.transpose(1, 2)) / p.sum(-1, keepdim=True)
    return out.flatten(1, 2).half()


def _count_pages(tables, keep, n_pages):
    keep = keep & (tables >= 0)
    index = torch.where(keep, tables, n_pages).long().flatten()
    return torch.zeros(n_pages + 1, dtype=torch.int32, device=tables.device).index_add_(0, index, torch.ones_like(index, dtype=torch.int32))[:n_pages]


def _take_pages(refs, wanted):
    """The lowest free pages, one for each true entry of `wanted` in order; -1 elsewhere. Their reference count becomes 1."""
    free = torch.nonzero(refs == 0).flatten().int()
    rank = torch.cumsum(wanted.int(), 0) - 1
    got = torch.where(wanted, free[rank.clamp_min(0)], -1)
    refs = refs.clone()
    refs[got[wanted].long()] = 1
    return got, refs


def _plain_fork(s):
    c = s["case"]
    tables, lens, refs, parents = s["tables"], s["lens"], s["refs"], s["parents"].long()
    n, page = refs.numel(), c["page"]
    col = torch.arange(tables.shape[1], device="cuda")[None, :]
    row = torch.arange(tables.shape[0], device="cuda")
    held = lambda ln: col < (ln[:, None] + page - 1) // page  # noqa: E731
    new_lens = lens[parents]
    new_tables = torch.where(held(new_lens), tables[parents], -1)
    first = ~((parents[:, None] == parents[None, :]) & (row[:, None] > row[None, :])).any(1)
    copied = ~first & (new_lens % page != 0)
    last = (new_lens.long() // page).clamp_max(tables.shape[1] - 1)
    src = torch.where(copied, new_tables[row, last], -1)
    refs = refs - _count_pages(tables, held(lens), n) + _count_pages(new_tables, held(new_lens) & ~(copied[:, None] & (col == last[:, None])), n)
    dst, refs = _take_pages(refs, copied)
    new_tables[row, last] = torch.where(copied, dst, new_tables[row, last])
    s["pool"][:, dst[copied].long()] = s["pool"][:, src[copied].long()]
    # room for one more token of every sequence
    grown = (new_lens % page == 0)
    got, refs = _take_pages(refs, grown)
    at = (new_lens.long() // page).clamp_max(tables.shape[1] - 1)
    new_tables[row, at] = torch.where(grown, got, new_tables[row, at])
    return new_tables, new_lens + s["add"], refs, src, dst, s["pool"]


def _plain_compact(s):
    tables, refs = s["tables"], s["refs"]
    n = refs.numel()
    live = refs > 0
    count = int(live.sum())
    page = torch.arange(n, device="cuda")
    src, dst = torch.nonzero(live & (page >= count)).flatten(), torch.nonzero(~live & (page < count)).flatten()
    remap = torch.where(live, page, -1).int()
    remap[src] = dst.int()
    new_refs = torch.where(page < count, refs, 0)
    new_refs[dst] = refs[src]
    s["pool"][:, dst] = s["pool"][:, src]
    return torch.where(tables >= 0, remap[tables.clamp_min(0).long()], -1), new_refs, remap, s["pool"]


def _plain_beam(s):
    c = s["case"]
    batch, beams, vocab = c["batch"], c["beams"], c["vocab"]
    x = s["logits"].double()                                             # candidates next to each other differ little
    top = x.amax(-1, keepdim=True)
    logp = x - top - torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    score = s["scores"].double()[:, None] + logp
    token = torch.arange(vocab, device="cuda")
    stay = torch.where(token == s["end"], s["scores"].double()[:, None], float("-inf"))
    score = torch.where(s["finished"][:, None], stay, score).view(batch, beams * vocab)
    best, index = torch.sort(score, dim=1, descending=True, stable=True)  # equal scores: the lowest index first
    best, index = best[:, :beams].flatten(), index[:, :beams]
    tokens = (index % vocab).int().flatten()
    parents = (index // vocab + beams * torch.arange(batch, device="cuda")[:, None]).int().flatten()
    p = parents.long()
    lens, done = s["lens"][p], s["finished"][p]
    col = torch.arange(c["history"], device="cuda")[None, :]
    history = torch.where(col < lens[:, None], s["history"][p], 0)
    history = torch.where((col == lens[:, None]) & ~done[:, None], tokens[:, None], history)
    return best.float(), tokens, parents, history, lens + (~done).int(), done | (tokens == s["end"])


def run(state):
    s, c = state, state["case"]
    if own:
        d = _device()
        if c["op"] == "rotary":
            q = d.rotary_paged(s["q"], s["k"], s["v"], s["positions"], s["seq_ids"], s["freq"], s["k_pages"], s["v_pages"], s["tables"],
                               layout=c["layout"], magnitude=s["magnitude"])
            return q, s["k_pages"], s["v_pages"]
        if c["op"] == "attention":
            return d.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["tables"], s["lens"], s["scale"], max_len=c["high"])
        if c["op"] == "fork":
            tables, lens, refs, src, dst, _ = d.pages_fork(s["tables"], s["lens"], s["refs"], s["parents"], c["page"])
            d.pages_copy(s["pool"], src, dst)
            d.pages_extend(tables, lens, refs, s["add"], c["page"])
            return tables, lens, refs, src, dst, s["pool"]
        if c["op"] == "compact":
            tables, refs, remap, src, dst, _ = d.pages_compact(s["tables"], s["refs"])
            d.pages_copy(s["pool"], src, dst)
            return tables, refs, remap, s["pool"]
        scores, tokens, parents = d.beam_select(s["logits"], s["scores"], c["beams"], finished=s["finished"], end_token=s["end"])
        history, lens, finished = d.beam_advance(s["history"], s["lens"], s["finished"], parents, tokens, end_token=s["end"])
        return scores, tokens, parents, history, lens, finished
    return {"rotary": _plain_rotary, "attention": _plain_attention, "fork": _plain_fork, "compact": _plain_compact, "beam": _plain_beam}[c["op"]](s)


# ------------------------------------------------------------------------------------------------ what a pass has to do

def work(case):
    c = case
    if c["op"] == "rotary":
        values = c["tokens"] * (c["heads"] + 2 * c["kv_heads"]) * c["dim"]
        return {"bytes": 4 * values + 12 * c["tokens"] + 4 * c["rotary"], "flops": 3 * c["tokens"] * (c["heads"] + c["kv_heads"]) * c["rotary"]}
    if c["op"] == "attention":
        total = int(_lengths(c["seqs"], c["low"], c["high"]).sum())
        pages = int(_pages_of(_lengths(c["seqs"], c["low"], c["high"]), c["page"]).sum())
        return {"bytes": 4 * total * c["kv_heads"] * c["dim"] + 4 * c["seqs"] * c["heads"] * c["dim"] + 4 * pages + 4 * c["seqs"],
                "flops": 4 * total * c["heads"] * c["dim"]}
    page_bytes = 2 * c.get("planes", 0) * c.get("page", 0) * c.get("kv_heads", 0) * c.get("dim", 0)
    if c["op"] == "fork":
        length = _lengths(c["requests"], max(2, c["length"] // 2), c["length"])
        copies = c["dropped"] * int((length % c["page"] != 0).sum())
        rows = c["requests"] * c["beams"]
        entries = c["beams"] * int(_pages_of(length, c["page"]).sum())
        return {"bytes": 2 * copies * page_bytes + 4 * (entries + rows * c["table"]) + 8 * entries + 28 * rows, "flops": 4 * entries}
    if c["op"] == "compact":
        # live pages lie anywhere in the pool: the share above the line moves
        moved = int(c["live"] * (1 - c["live"] / c["pages"]))
        return {"bytes": 2 * moved * page_bytes + 8 * c["seqs"] * c["table"] + 12 * c["pages"], "flops": 2 * c["pages"]}
    rows = c["batch"] * c["beams"]
    return {"bytes": 2 * rows * c["vocab"] + 8 * rows * c["history"] + 38 * rows, "flops": 4 * rows * c["vocab"]}


# ------------------------------------------------------------------------------------------------ by definition, in 64 bits

def exact(case, seed):
    c, s = case, prepare(case, seed)
    page = c.get("page", 1)
    if c["op"] == "rotary":
        # every pair as one complex number, turned by exp(i angle)
        turn = torch.polar(torch.full((1, 1), s["magnitude"], dtype=torch.float64, device="cuda"),
                           torch.outer(s["positions"].double(), s["freq"]))[:, None, :]
        half = s["freq"].numel()

        def rotated(x):
            x = x.double().clone()
            at = (slice(0, half), slice(half, 2 * half)) if c["layout"] == "half" else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
            z = torch.complex(x[..., at[0]], x[..., at[1]]) * turn
            x[..., at[0]], x[..., at[1]] = z.real, z.imag
            return x

        flat = s["seq_ids"].long() * s["tables"].shape[1] + torch.div(s["positions"], page, rounding_mode="floor").long()
        slot = s["tables"].flatten()[flat].long() * page + s["positions"].long() % page
        k_pages, v_pages = s["k_pages"].double().flatten(0, 1), s["v_pages"].double().flatten(0, 1)
        k_pages[slot], v_pages[slot] = rotated(s["k"]), s["v"].double()
        return rotated(s["q"]), k_pages.view(s["k_pages"].shape), v_pages.view(s["v_pages"].shape)
    if c["op"] == "attention":
        out = []
        for i, n in enumerate(s["lens"].tolist()):
            rows = s["tables"][i, : -(-n // page)].long()
            k, v = (t[rows].flatten(0, 1)[:n].double() for t in (s["k_pages"], s["v_pages"]))      # [n, kv heads, dim]
            q = s["q"][i].double().view(c["kv_heads"], -1, c["dim"])
            score = s["scale"] * torch.stack([q[h] @ k[:, h].t().contiguous() for h in range(c["kv_heads"])])
            out.append(torch.stack([torch.softmax(score[h], -1) @ v[:, h].contiguous() for h in range(c["kv_heads"])]).flatten(0, 1))
        return torch.stack(out)
    if c["op"] == "fork":
        tables, lens, refs, parents = (s[k].tolist() for k in ("tables", "lens", "refs", "parents"))
        width, rows = c["table"], len(parents)
        for i in range(rows):
            for p in tables[i][: -(-lens[i] // page)]:
                refs[p] -= 1
        new, src, dst, seen, new_lens = [], [-1] * rows, [-1] * rows, set(), [lens[p] for p in parents]
        for i, p in enumerate(parents):
            used = -(-lens[p] // page)
            new.append(tables[p][:used] + [-1] * (width - used))
            if p in seen and lens[p] % page:
                src[i] = new[i][used - 1]
            for j in range(used - (src[i] >= 0)):
                refs[new[i][j]] += 1
            seen.add(p)
        for i in range(rows):
            if src[i] >= 0:
                dst[i] = refs.index(0)
                refs[dst[i]] = 1
                new[i][new_lens[i] // page] = dst[i]
                s["pool"][:, dst[i]] = s["pool"][:, src[i]]
        for i in range(rows):
            if new_lens[i] % page == 0:
                new[i][new_lens[i] // page] = refs.index(0)
                refs[refs.index(0)] = 1
        ints = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (new, [n + 1 for n in new_lens], refs, src, dst)]
        return (*ints, s["pool"])
    if c["op"] == "compact":
        tables, refs = s["tables"].tolist(), s["refs"].tolist()
        remap, count = [p if r else -1 for p, r in enumerate(refs)], sum(r > 0 for r in refs)
        holes = iter([p for p in range(count) if not refs[p]])
        for p in range(count, len(refs)):
            if refs[p]:
                hole = next(holes)
                remap[p], refs[hole], refs[p] = hole, refs[p], 0
                s["pool"][:, hole] = s["pool"][:, p]
        tables = [[remap[p] if p >= 0 else -1 for p in row] for row in tables]
        ints = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (tables, refs, remap)]
        return (*ints, s["pool"])
    out = [[], [], [], [], [], []]
    logp = torch.log_softmax(s["logits"].double(), -1) + s["scores"].double()[:, None]
    history, lens, finished, scores = s["history"].tolist(), s["lens"].tolist(), s["finished"].tolist(), s["scores"].double().tolist()
    for b in range(c["batch"]):
        found = []
        for r in range(b * c["beams"], (b + 1) * c["beams"]):
            if finished[r]:
                found.append((-scores[r], r, s["end"]))
                found += [(math.inf, r, t) for t in range(c["beams"] + 1) if t != s["end"]]
                continue
            row = logp[r]
            bound = torch.topk(row, min(c["beams"], c["vocab"])).values[-1]
            found += [(-float(row[t]), r, t) for t in torch.nonzero(row >= bound).flatten().tolist()]
        for neg, r, t in sorted(found)[: c["beams"]]:
            line = history[r][: lens[r]] + ([] if finished[r] else [t])
            values = (-neg, t, r, (line + [0] * c["history"])[: c["history"]], len(line), finished[r] or t == s["end"])
            for to, x in zip(out, values):
                to.append(x)
    types = (torch.float64, torch.int32, torch.int32, torch.int32, torch.int32, torch.bool)
    return tuple(torch.tensor(x, dtype=t, device="cuda") for x, t in zip(out, types))
