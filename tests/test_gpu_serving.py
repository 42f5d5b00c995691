"""GPU parity of the serving operators (rotary, paged attention, page bookkeeping, beam search) against their definitions
in 64 bits, through the public entry points. Integers and copies are compared exactly.

Tolerances, from the arithmetic: a rounding to half is off by 2^-11 of the value, or 2^-25 where it is subnormal.
  rotary     sine and cosine come from an angle rounded to 2^-25 turns (2e-7 rad) by a function good to 2 ulp (2.4e-7), times
             the magnitude, and two products and a sum of fp32 (3 * 2^-24): together below 8e-7 (|a| + |b|) magnitude.
  attention  a score is a sum of D exact products in fp32: off by at most D 2^-24 scale sum|q k|; its exponential by as much
             again relatively, plus 2^-19 for the exponent's own rounding (|s| log2 e up to 2^7 at 2^-24, with the two
             roundings of the running maximum) and the exponential; it enters once above and once below the line of
             the quotient. Sums run through at most 1024 fp32 additions one after the other.
  beam       a row's sum of exponentials good to 2^-22 moves the logarithm by 2^-22; the result is rounded to fp32."""
import math

import numpy as np
import pytest
import torch

from tensorlib_amd import TensorLibError

pytestmark = pytest.mark.gpu


def rand(shape, seed, std=1.0, dtype=torch.float16):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * std).to(dtype)


def ints(a):
    return torch.as_tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def within(got, want, slack, what):
    got, want = got.double(), want.double()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), f"{what}: NaN in other places"
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), f"{what}: infinities differ"
    tol = torch.maximum(want.abs() * 2.0 ** -11, torch.full_like(want, 2.0 ** -25)) + slack
    off = ((got - want).abs() > tol) & ~nan & ~inf
    assert not off.any(), f"{what}: {int(off.sum())} of {off.numel()} off, worst {float(((got - want).abs() / tol)[~nan & ~inf].max())} times the tolerance"


# ------------------------------------------------------------------------------------------------ rotary

def rotated(x, positions, freq, layout, magnitude):
    """In 64 bits, and the scale of each element's error: |a| + |b| of its pair (0 where it is copied)."""
    x, half = x.double(), freq.numel()
    out, size = x.clone(), torch.zeros_like(x)
    angle = (positions.double()[:, None] * freq[None, :])[:, None, :]
    ia = slice(0, half) if layout == "half" else slice(0, 2 * half, 2)
    ib = slice(half, 2 * half) if layout == "half" else slice(1, 2 * half, 2)
    a, b = x[..., ia], x[..., ib]
    out[..., ia] = magnitude * (a * angle.cos() - b * angle.sin())
    out[..., ib] = magnitude * (a * angle.sin() + b * angle.cos())
    size[..., ia] = size[..., ib] = (a.abs() + b.abs()) * abs(magnitude)
    return out, size


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("n,h,d,rd", [(1, 32, 128, 128), (3, 1, 64, 32), (257, 3, 128, 128), (65, 5, 80, 20), (33, 2, 256, 64), (7, 4, 96, 96), (5, 3, 2, 2),
                                      (9, 2, 7, 4), (4, 2, 33, 32), (6, 3, 64, 0), (1000, 8, 64, 64), (2, 7, 40, 8), (4101, 9, 128, 64)])
def test_rotary(dev, layout, n, h, d, rd):
    x = rand((n, h, d), 1)
    rng = np.random.RandomState(n)
    positions = ints(rng.randint(0, 200000, n))
    freq = dev.rotary_frequencies(rd) if rd else torch.empty(0, dtype=torch.float64, device="cuda")
    want, size = rotated(x, positions, freq, layout, 1.25)
    got = dev.rotary(x, positions, freq, layout, 1.25)
    within(got, want, 8e-7 * size, "rotary")
    assert torch.equal(got[..., rd:], x[..., rd:])
    y = x.clone()
    dev.rotary(y, positions, freq, layout, 1.25, out=y)
    assert torch.equal(y, got), "in place"
    wide = rand((n, 3 * h * d + 8), 2)                       # a column block of a wider matrix, into another
    wide[:, 8: 8 + h * d] = x.flatten(1)
    into = torch.full((n, 2 * h * d), 7.0, dtype=torch.float16, device="cuda")
    dev.rotary(wide[:, 8: 8 + h * d].unflatten(1, (h, d)), positions, freq, layout, 1.25, out=into[:, h * d:].unflatten(1, (h, d)))
    assert torch.equal(into[:, h * d:], got.flatten(1)) and bool((into[:, : h * d] == 7.0).all())
    odd = torch.empty(n * h * d + 1, dtype=torch.float16, device="cuda")[1:].view(n, h, d)      # 2-byte aligned only
    odd.copy_(x)
    within(dev.rotary(odd, positions, freq, layout, 1.25), want, 8e-7 * size, "rotary, misaligned")


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("offset,row,h,d,rd", [(0, 0, 3, 80, 20), (2, 0, 2, 64, 64), (4, 4, 2, 64, 64), (4, 2, 3, 96, 24), (0, 4, 3, 40, 40), (6, 8, 2, 128, 64),
                                               (8, 12, 2, 16, 16), (0, 2, 1, 12, 8), (2, 6, 5, 10, 4), (1, 8, 2, 32, 32), (8, 1, 2, 32, 32), (4, 0, 7, 20, 12)])
def test_rotary_at_every_alignment(dev, layout, offset, row, h, d, rd):
    """Elements that the first row and the rows after it are off a multiple of 16 bytes, in and out; what lies around the rows
    stays."""
    n, width = 67, (h * d + 7) // 8 * 8 + 8
    x, out = (rand(n * (width + row) + 16, s) for s in (1, 2))
    view = lambda t: torch.as_strided(t, (n, h, d), (width + row, d, 1), offset)  # noqa: E731
    positions = ints(np.random.RandomState(d).randint(0, 100000, n))
    freq = dev.rotary_frequencies(rd)
    want, size = rotated(view(x), positions, freq, layout, 1.0)
    kept = out.clone()
    dev.rotary(view(x), positions, freq, layout, out=view(out))
    within(view(out), want, 8e-7 * size, "rotary")
    view(kept).copy_(view(out))
    assert torch.equal(out, kept)


@pytest.mark.parametrize("n,h,kv,d,rd,layout", [(3000, 8, 8, 96, 24, "half"), (3000, 8, 8, 80, 20, "half"), (3000, 9, 8, 80, 80, "half"), (3000, 8, 8, 96, 96, "half"), (3000, 8, 8, 80, 20, "interleaved"),
                                               (2000, 32, 2, 64, 64, "interleaved"), (29000, 8, 8, 96, 96, "half"), (22000, 9, 8, 128, 128, "half"), (22000, 8, 8, 128, 64, "interleaved"),
                                               (35000, 8, 8, 80, 40, "half")])
def test_rotary_of_many_tokens(dev, n, h, kv, d, rd, layout):
    """Large batches move their values otherwise, and compute the same."""
    page, step = 16, 1000
    q, k, v = rand((n, h, d), 1), rand((n, kv, d), 2), rand((n, kv, d), 3)
    positions, n_pages = torch.arange(n, dtype=torch.int32, device="cuda"), -(-n // page)
    tables = torch.randperm(n_pages, generator=torch.Generator().manual_seed(1)).int().cuda()[None]
    seq_ids = torch.zeros(n, dtype=torch.int32, device="cuda")
    freq = dev.rotary_frequencies(rd)
    kp, vp = (torch.zeros((n_pages, page, kv, d), dtype=torch.float16, device="cuda") for _ in range(2))
    got = dev.rotary_paged(q, k, v, positions, seq_ids, freq, kp, vp, tables, layout)
    for a in range(0, n, step):                                        # small calls, checked above
        part = slice(a, a + step)
        assert torch.equal(got[part], dev.rotary(q[part], positions[part], freq, layout)), a
        rows = positions[part].long()
        pages = tables[0][rows // page].long()
        assert torch.equal(kp[pages, rows % page], dev.rotary(k[part], positions[part], freq, layout)) and torch.equal(vp[pages, rows % page], v[part]), a


def test_rotary_far_negative_and_special_values(dev):
    n, h, d = 6, 2, 64
    x = rand((n, h, d), 3)
    positions = ints([0, -1, 2 ** 31 - 1, -2 ** 31, 10 ** 9 + 7, 1])
    freq = dev.rotary_frequencies(d, base=500000.0, scaling="parts", factor=4.0, original_context=8192.0)
    for layout in ("half", "interleaved"):
        want, size = rotated(x, positions, freq, layout, 1.0)
        # 2^31 positions of up to 1 rad: the fp64 product and its factor 1 / 2 pi leave 2^31 * 3 * 2^-53 rad more
        within(dev.rotary(x, positions, freq, layout), want, (8e-7 + 8e-7) * size, "far positions")
    y = x.clone()
    y[0, 0, 5], y[1, 1, 6], y[2, 0, 7] = float("nan"), float("inf"), 65504.0
    got = dev.rotary(y, positions, freq, "interleaved")
    clean = dev.rotary(x, positions, freq, "interleaved")
    same = torch.ones_like(clean, dtype=torch.bool)
    for a, b, c in ((0, 0, 4), (0, 0, 5), (1, 1, 6), (1, 1, 7), (2, 0, 6), (2, 0, 7)):      # the pairs that hold them
        same[a, b, c] = False
    assert torch.equal(got[same], clean[same])
    assert torch.isnan(got[0, 0, 4]) and torch.isnan(got[0, 0, 5]) and not torch.isfinite(got[1, 1, 6:8]).any()
    assert dev.rotary(x[:0], positions[:0], freq).shape == (0, h, d)


def paged_cache(n_pages, page, kv, d, order, seed=11):
    """(k, v) as [pages, positions, heads, dim] in either memory order."""
    shape = (n_pages, page, kv, d) if order == "row" else (n_pages, kv, page, d)
    k, v = rand(shape, seed), rand(shape, seed + 1)
    return (k, v) if order == "row" else (k.permute(0, 2, 1, 3), v.permute(0, 2, 1, 3))


@pytest.mark.parametrize("order", ["row", "head"])
@pytest.mark.parametrize("layout,h,kv,d,rd,page", [("half", 8, 2, 128, 128, 16), ("interleaved", 4, 4, 64, 64, 16), ("half", 6, 1, 80, 20, 3), ("interleaved", 3, 3, 96, 24, 1),
                                                   ("half", 2, 2, 256, 128, 24), ("interleaved", 5, 5, 8, 4, 7), ("half", 0, 2, 64, 64, 8)])
def test_rotary_paged(dev, order, layout, h, kv, d, rd, page):
    starts, news = [0, 5, 37, 1000], [9, 1, 70, 2]                     # ragged sequences, some begun earlier
    n = sum(news) + 2
    seq_ids = np.concatenate([np.full(c, i) for i, c in enumerate(news)] + [[-1, 4]])       # padded, and no such sequence
    positions = np.concatenate([np.arange(a, a + c) for a, c in zip(starts, news)] + [[3, 3]])
    width = -(-max(a + c for a, c in zip(starts, news)) // page)
    n_pages = 4 * width + 3
    tables = np.random.RandomState(5).permutation(n_pages)[: 4 * width].reshape(4, width)
    qkv = rand((n, (h + 2 * kv) * d + 8), 6)
    q, k, v = (qkv[:, a: a + c * d].unflatten(1, (c, d)) for a, c in ((0, h), (h * d, kv), ((h + kv) * d, kv)))
    kp, vp = paged_cache(n_pages, page, kv, d, order)
    k0, v0 = kp.clone(), vp.clone()
    freq = dev.rotary_frequencies(rd, scaling="linear", factor=4.0)
    got = dev.rotary_paged(q, k, v, ints(positions), ints(seq_ids), freq, kp, vp, ints(tables), layout, 1.0)
    want, size = rotated(q, ints(positions), freq, layout, 1.0)
    within(got, want, 8e-7 * size, "q")
    kr = dev.rotary(k, ints(positions), freq, layout)                  # checked above
    for t in range(n - 2):
        p, r = int(tables[seq_ids[t], positions[t] // page]), int(positions[t] % page)
        k0[p, r], v0[p, r] = kr[t], v[t]
    assert torch.equal(kp, k0) and torch.equal(vp, v0), "cache rows, and nothing beside them"


def test_rotary_paged_leaves_out_what_has_no_place(dev):
    kv, d, page, n_pages = 2, 64, 16, 6
    kp, vp = paged_cache(n_pages, page, kv, d, "row")
    k0, v0 = kp.clone(), vp.clone()
    tables = ints([[0, -1, 6], [2 ** 31 - 1, 4, 5]])
    q = rand((6, 4, d), 1)
    k = rand((6, kv, d), 2)
    # an empty entry, a page past the pool, a position past the table, a negative one, another past the pool, a good one
    positions, seq_ids = ints([16, 40, 48, -1, 3, 20]), ints([0, 0, 0, 0, 1, 1])
    freq = dev.rotary_frequencies(d)
    dev.rotary_paged(q, k, k, positions, seq_ids, freq, kp, vp, tables)
    k0[4, 4], v0[4, 4] = dev.rotary(k, positions, freq)[5], k[5]
    assert torch.equal(kp, k0) and torch.equal(vp, v0)
    one = dev.rotary_paged(q[:2], k[:2], k[:2], ints([1, 17]), None, freq, kp, vp, tables)       # token i is of sequence i
    k0[0, 1], v0[0, 1] = dev.rotary(k[:1], ints([1]), freq)[0], k[0]
    k0[4, 1], v0[4, 1] = dev.rotary(k[1:2], ints([17]), freq)[0], k[1]
    assert torch.equal(kp, k0) and torch.equal(vp, v0) and one.shape == (2, 4, d)


# ------------------------------------------------------------------------------------------------ attention

def attention(q, kp, vp, tables, lens, scale):
    """By definition in 64 bits; and the slack that the fp32 steps need, from the data."""
    b, h, d = q.shape
    _, page, kv, _ = kp.shape
    out, slack = torch.zeros(b, h, d, dtype=torch.float64, device="cuda"), torch.zeros(b, h, d, dtype=torch.float64, device="cuda")
    for i, n in enumerate(lens):
        if n <= 0:
            continue
        pages = torch.as_tensor(tables[i][: -(-n // page)], device="cuda").long()
        k, v = (t[pages].flatten(0, 1)[:n].double().transpose(0, 1).contiguous() for t in (kp, vp))        # [kv, n, d]
        qi = q[i].double().view(kv, h // kv, d)
        s = scale * torch.matmul(qi, k.transpose(1, 2).contiguous())
        p = torch.softmax(s, -1)
        out[i] = torch.matmul(p, v).flatten(0, 1)
        size = abs(scale) * torch.matmul(qi.abs(), k.abs().transpose(1, 2).contiguous()).nan_to_num().amax(-1, keepdim=True)
        delta = 2 * (2.0 ** -19 + d * 2.0 ** -24 * size) + 2 * 1024 * 2.0 ** -24
        slack[i] = (delta * torch.matmul(p.nan_to_num(), v.abs().nan_to_num())).flatten(0, 1)
    return out, slack


def tables_for(lens, page, n_extra=3, seed=3, width=None):
    rng = np.random.RandomState(seed)
    used = [max(0, -(-n // page)) for n in lens]
    width = width or max(max(used), 1)
    n_pages = sum(used) + n_extra
    order = rng.permutation(n_pages)
    t = np.full((len(lens), width), -1, np.int64)
    at = 0
    for i, u in enumerate(used):
        t[i, :u] = order[at: at + u]
        at += u
    return t, n_pages


def spoil_unused(kp, vp, tables, lens):
    """Everything that no sequence covers becomes NaN or infinite: none of it may show."""
    page = kp.shape[1]
    keep = torch.zeros(kp.shape[:2], dtype=torch.bool, device="cuda")
    for i, n in enumerate(lens):
        for c in range(max(0, -(-n // page))):
            keep[int(tables[i, c]), : min(page, n - c * page)] = True
    kp[~keep] = float("nan")
    vp[~keep] = float("nan")
    vp[~keep & (torch.arange(page, device="cuda") % 2 == 0)] = float("inf")


@pytest.mark.parametrize("order", ["row", "head"])
@pytest.mark.parametrize("h,kv,d,page", [(32, 32, 128, 16), (32, 8, 128, 16), (8, 1, 64, 1), (6, 2, 80, 20), (16, 1, 128, 24), (17, 1, 64, 16), (40, 1, 96, 8), (66, 2, 256, 32),
                                         (4, 4, 8, 3), (10, 5, 136, 64), (64, 4, 128, 256), (2, 2, 256, 16), (3, 1, 40, 5), (9, 3, 248, 16)])
def test_paged_attention(dev, order, h, kv, d, page):
    lens = [1, 0, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 300, 1025]
    tables, n_pages = tables_for(lens, page)
    kp, vp = paged_cache(n_pages, page, kv, d, order)
    spoil_unused(kp, vp, tables, lens)
    q = rand((len(lens), h, d), 8)
    want, slack = attention(q, kp, vp, tables, lens, 0.1)
    got = dev.paged_attention(q, kp, vp, ints(tables), ints(lens), 0.1)
    within(got, want, slack, "attention")
    # the same through the short bound alone (one pass or a few chunks), and with queries inside wider rows
    wide = rand((len(lens), h * d + 24), 9)
    wide[:, 8: 8 + h * d] = q.flatten(1)
    got = dev.paged_attention(wide[:, 8: 8 + h * d].unflatten(1, (h, d)), kp, vp, ints(tables), ints(lens), 0.1, max_len=1025)
    within(got, want, slack, "attention, strided")


@pytest.mark.parametrize("b,h,kv,d,page,low,high", [(1, 32, 32, 128, 16, 2048, 2048), (1, 8, 8, 128, 16, 20000, 20000), (2, 64, 8, 128, 64, 9000, 33333), (200, 8, 1, 64, 16, 1, 400),
                                                    (1, 16, 1, 128, 128, 131072, 131072), (3, 4, 4, 256, 8, 777, 5001), (64, 32, 32, 64, 16, 1, 3000)])
def test_paged_attention_long_and_many(dev, b, h, kv, d, page, low, high):
    rng = np.random.RandomState(1)
    lens = rng.randint(low, high + 1, b)
    lens[0] = high
    tables, n_pages = tables_for(lens, page)
    kp, vp = paged_cache(n_pages, page, kv, d, "row")
    q = rand((b, h, d), 8)
    want, slack = attention(q, kp, vp, tables, lens, 1 / math.sqrt(d))
    got = dev.paged_attention(q, kp, vp, ints(tables), ints(lens), max_len=high)
    within(got, want, slack, "attention")
    assert torch.equal(got, dev.paged_attention(q, kp, vp, ints(tables), ints(lens), max_len=high)), "not the same twice"


def test_paged_attention_special_values(dev):
    """Outliers far above the rest, scores of -inf, infinities in the values, whole rows of -inf, and NaN where it belongs."""
    h, kv, d, page, lens = 4, 2, 64, 16, [100, 100, 100, 100, 700]
    tables, n_pages = tables_for(lens, page)
    kp, vp = paged_cache(n_pages, page, kv, d, "row")
    q = rand((5, h, d), 8)
    q[:, :, 0] = 1.0
    at = lambda i, t: (int(tables[i, t // page]), t % page)  # noqa: E731
    kp[at(0, 40)][0, 0] = 30000.0                                  # one position outweighs all others of kv head 0
    kp[at(0, 40)][1, 0] = -30000.0                                 # and has no weight for kv head 1
    kp[at(1, 3)][0, 0] = float("-inf")                             # a score of -inf
    vp[at(1, 70)][1, 5] = float("inf")
    vp[at(1, 71)][0, 6] = float("-inf")
    for t in range(100):
        kp[at(2, t)][1, 0] = float("-inf")                         # no position left for kv head 1: 0 / 0
    kp[at(3, 50)][0, 3] = float("nan")
    kp[at(4, 650)][0, 0] = 20000.0                                 # the maximum comes late
    for t in range(0, 256):
        kp[at(4, t)][1, 0] = float("-inf")                         # the first chunks of kv head 1 are all -inf
    want, slack = attention(q, kp, vp, tables, lens, 0.125)
    assert torch.isnan(want[2, 2:]).all() and torch.isnan(want[3, :2]).all() and torch.isfinite(want[4]).all()
    got = dev.paged_attention(q, kp, vp, ints(tables), ints(lens), 0.125)
    within(got, want, slack, "special values")
    for scale in (0.0, -0.3, 40.0):
        want, slack = attention(q[4:], kp, vp, tables[4:], lens[4:], scale) if scale > 0 else attention(q[4:, :2], kp[:, :, :1], vp[:, :, :1], tables[4:], lens[4:], scale)
        got = (dev.paged_attention(q[4:], kp, vp, ints(tables[4:]), ints(lens[4:]), scale) if scale > 0 else
               dev.paged_attention(q[4:, :2], kp[:, :, :1], vp[:, :, :1], ints(tables[4:]), ints(lens[4:]), scale))
        within(got, want, slack, f"scale {scale}")


def test_paged_attention_bad_tables_answer_nan_for_their_sequence_alone(dev):
    h, kv, d, page = 4, 2, 64, 16
    lens = [50, 50, 50, 3000, 50, 200, -7]
    tables, n_pages = tables_for(lens, page)
    tables[1, 2], tables[2, 0], tables[3, 100] = -1, n_pages, 2 ** 31 - 1
    kp, vp = paged_cache(n_pages, page, kv, d, "row")
    q = rand((len(lens), h, d), 8)
    good = [0, 4, 5, 6]
    want, slack = attention(q[good], kp, vp, tables[good], [lens[i] for i in good], 0.125)
    for max_len in (None, 3000):
        got = dev.paged_attention(q, kp, vp, ints(tables), ints(lens), 0.125, max_len=max_len)
        within(got[good], want, slack, "good sequences")
        assert torch.isnan(got[1:4]).all() and bool((got[6] == 0).all())
    got = dev.paged_attention(q, kp, vp, ints(tables), ints(lens), 0.125, max_len=100)         # lens beyond the bound
    assert torch.isnan(got[3]).all() and torch.isnan(got[5]).all()
    within(got[[0, 4]], want[:2], slack[:2], "below the bound")
    got = dev.paged_attention(q, kp, vp, ints(tables[:, :10]), ints(lens), 0.125, max_len=3000)     # and beyond the table
    assert torch.isnan(got[3]).all() and torch.isnan(got[5]).all()
    within(got[[0, 4]], want[:2], slack[:2], "inside the table")
    assert bool((dev.paged_attention(q, kp, vp, ints(tables), ints([0] * 7), 0.125) == 0).all())


def test_offsets_past_32_bits(dev):
    """Pages whose elements lie 2^32 and more elements behind the first (a pool of 9 GB for each of k and v)."""
    kv, d, page = 1, 64, 16
    stride = 1 << 21                                               # elements between pages
    n_pages = (1 << 32) // stride + 3
    big = torch.empty(2 * (n_pages * stride), dtype=torch.float16, device="cuda")
    kp, vp = (t.as_strided((n_pages, page, kv, d), (stride, kv * d, d, 1)) for t in (big[: n_pages * stride], big[n_pages * stride:]))
    lens, far = [40, 16], [n_pages - 1, 3, n_pages - 2]
    tables = np.array([far, [1024, -1, -1]])
    for p in far + [1024]:
        kp[p], vp[p] = rand((page, kv, d), 20 + p % 7), rand((page, kv, d), 30 + p % 7)
    q = rand((2, 4, d), 8)
    want, slack = attention(q, kp, vp, tables, lens, 0.125)
    within(dev.paged_attention(q, kp, vp, ints(tables), ints(lens), 0.125), want, slack, "far pages")
    k = rand((2, kv, d), 40)
    freq = dev.rotary_frequencies(d)
    dev.rotary_paged(q, k, k, ints([39, 2]), None, freq, kp, vp, ints(tables))
    kr = dev.rotary(k, ints([39, 2]), freq)
    assert torch.equal(kp[n_pages - 2, 7, 0], kr[0, 0]) and torch.equal(vp[1024, 2, 0], k[1, 0])
    pool = big.view(2, n_pages, stride)[:, :, :1024]               # a page's bytes, planes 2^33 bytes apart
    dev.pages_copy(pool, ints([n_pages - 1, 1024]), ints([0, n_pages - 3]))
    assert torch.equal(pool[:, 0], pool[:, n_pages - 1]) and torch.equal(pool[:, n_pages - 3], pool[:, 1024])


# ------------------------------------------------------------------------------------------------ pages

def fork_by_hand(tables, lens, refs, parents, page):
    """The definition in plain loops; None if pages are lacking."""
    tables, lens, refs = [list(map(int, r)) for r in tables], list(map(int, lens)), list(map(int, refs))
    width, n = len(tables[0]), len(tables)
    pages = lambda ln: min(-(-ln // page), width)  # noqa: E731
    for i in range(n):
        for p in tables[i][: pages(lens[i])]:
            if 0 <= p < len(refs):
                refs[p] -= 1
    new, new_lens, src, dst, seen = [], [], [-1] * n, [-1] * n, set()
    for i, parent in enumerate(parents):
        parent = int(parent)
        ln = lens[parent] if 0 <= parent < n else 0
        row = (tables[parent][: pages(ln)] if ln else []) + [-1] * (width - pages(ln))
        if parent in seen and ln % page and 0 <= row[pages(ln) - 1] < len(refs):
            src[i] = row[pages(ln) - 1]
        for c in range(pages(ln) - (src[i] >= 0)):
            if 0 <= row[c] < len(refs):
                refs[row[c]] += 1
        if ln:
            seen.add(parent)
        new.append(row)
        new_lens.append(ln)
    if refs.count(0) < sum(s >= 0 for s in src):
        return None
    for i in range(n):
        if src[i] >= 0:
            dst[i] = refs.index(0)
            refs[dst[i]] = 1
            new[i][pages(new_lens[i]) - 1] = dst[i]
    return new, new_lens, refs, src, dst


def state(rows, page, width, seed, spare, lens=None):
    rng = np.random.RandomState(seed)
    lens = rng.randint(0, page * width + 1, rows) if lens is None else np.asarray(lens)
    tables, n_pages = tables_for(lens, page, spare, seed, width)
    refs = np.bincount(tables[tables >= 0], minlength=n_pages)
    return tables, lens, refs, rng


@pytest.mark.parametrize("rows,page,width,spare", [(1, 16, 4, 2), (4, 16, 8, 8), (7, 5, 3, 20), (64, 16, 40, 70), (300, 8, 9, 400), (1100, 8, 5, 1500), (3, 1, 50, 9), (130, 16, 300, 5000), (40, 1, 2000, 90000)])
def test_fork_and_extend(dev, rows, page, width, spare):
    tables, lens, refs, rng = state(rows, page, width, rows, spare)
    parents = rng.randint(0, rows, rows)
    parents[rng.rand(rows) < 0.1] = -1
    for step in range(3):                                          # forks of forks: shared pages, freed pages
        want = fork_by_hand(tables, lens, refs, parents, page)
        before = [ints(a) for a in (tables, lens, refs)]
        kept = [t.clone() for t in before]
        *got, missing = dev.pages_fork(*before, ints(parents), page)
        assert all(torch.equal(a, b) for a, b in zip(before, kept)), "the old state changed"
        if want is None:
            assert int(missing) > 0 and all(torch.equal(a, b) for a, b in zip(got[:3], kept))
            assert bool((got[3] == -1).all()) and bool((got[4] == -1).all())
        else:
            assert int(missing) == 0
            for g, w, name in zip(got, want, ("tables", "lens", "refs", "src", "dst")):
                assert g.cpu().tolist() == [list(map(int, r)) for r in w] if name == "tables" else g.cpu().tolist() == list(map(int, w)), (name, step)
        tables, lens, refs = got[0].cpu().numpy(), got[1].cpu().numpy(), got[2].cpu().numpy()
        # room for more: by hand, page by page in row order
        add = rng.randint(0, 2 * page + 1, rows)
        add = np.where(lens + add <= page * width, add, 0)
        t, ln, r = ints(tables), ints(lens), ints(refs)
        wt, wr = tables.copy(), refs.copy()
        need = [(i, c) for i in range(rows) for c in range(-(-int(lens[i]) // page), -(-int(lens[i] + add[i]) // page))]
        free = np.flatnonzero(wr == 0)
        missing = dev.pages_extend(t, ln, r, ints(add), page)
        assert int(missing) == max(0, len(need) - len(free))
        if len(need) <= len(free):
            for (i, c), p in zip(need, free):
                wt[i, c], wr[p] = p, 1
            lens = lens + add
        assert np.array_equal(t.cpu().numpy(), wt) and np.array_equal(r.cpu().numpy(), wr) and np.array_equal(ln.cpu().numpy(), lens)
        tables, refs = wt, wr
        parents = rng.randint(-1, rows, rows)


@pytest.mark.parametrize("rows,width,n_pages", [(1, 9000, 9001), (3, 3000, 16384), (1024, 32, 16384), (1024, 31, 16385), (8192, 3, 30000), (8192, 2, 16383), (2, 8192, 16385),
                                                (65, 127, 8200)])
def test_extend_by_prompts_and_fork(dev, rows, width, n_pages):
    """Room for whole prompts at once, up to more pages than are listed on the way, and forks of what came of it, at the limits of
    a workgroup's shared memory."""
    page = 2
    rng = np.random.RandomState(rows + width)
    refs = (rng.rand(n_pages) < 0.05).astype(int)                  # pages that somebody else holds
    tables, lens = np.full((rows, width), -1), np.zeros(rows, int)
    for most in (1, width, width):
        free = np.flatnonzero(refs == 0)
        room = width - -(-lens // page)
        need = np.minimum(rng.randint(0, most + 1, rows), room)
        if rows == 1:
            need[:] = np.minimum(room, most)
        while need.sum() > len(free):
            need = need // 2
        add = np.where(need > 0, need * page - (-lens % page > 0) - rng.randint(0, 2, rows), 0)
        add = np.where(-(-(lens + add) // page) - -(-lens // page) == need, add, need * page)
        need = -(-(lens + add) // page) - -(-lens // page)
        t, ln, r = ints(tables), ints(lens), ints(refs)
        assert int(dev.pages_extend(t, ln, r, ints(add), page)) == 0
        ranks = np.cumsum(need) - need
        for i in range(rows):
            held = -(-int(lens[i]) // page)
            tables[i, held:held + need[i]] = free[ranks[i]:ranks[i] + need[i]]
        refs[free[:need.sum()]] = 1
        lens = lens + add
        assert np.array_equal(t.cpu().numpy(), tables) and np.array_equal(r.cpu().numpy(), refs) and np.array_equal(ln.cpu().numpy(), lens)
    parents = np.where(rng.rand(rows) < 0.3, np.arange(rows), rng.randint(-1, rows, rows))
    want = fork_by_hand(tables, lens, refs, parents, page)
    *got, missing = dev.pages_fork(t, ln, r, ints(parents), page)
    assert (want is None) == (int(missing) > 0)
    if want is not None:
        assert np.array_equal(got[0].cpu().numpy(), np.array(want[0]))
        assert all(np.array_equal(g.cpu().numpy(), np.array(w)) for g, w in zip(got[1:], want[1:]))


def test_fork_edges(dev):
    # parents out of range leave empty rows; a page counted by nobody's table stays; entries out of range are passed through
    page = 4
    tables = np.array([[0, 1, -1], [2, -1, -1], [3, 9, -1]])
    lens, refs = [6, 4, 5], [1, 1, 1, 1, 2, 0, 0]
    for parents in ([0, 0, 0], [5, -3, 1], [1, 1, 1], [2, 2, 2], [2, 0, 2]):
        want = fork_by_hand(tables, lens, refs, parents, page)
        *got, missing = dev.pages_fork(ints(tables), ints(lens), ints(refs), ints(parents), page)
        assert int(missing) == 0
        assert [g.cpu().tolist() for g in got] == [list(map(list, want[0])), *map(list, want[1:])], parents
    # three copies wanted, two pages free: nothing changes
    tables, lens, refs = np.array([[0], [-1], [-1], [-1]]), [3, 0, 0, 0], [1, 0, 0]
    *got, missing = dev.pages_fork(ints(tables), ints(lens), ints(refs), ints([0, 0, 0, 0]), page)
    assert int(missing) == 1 and [g.cpu().tolist() for g in got] == [tables.tolist(), lens, refs, [-1] * 4, [-1] * 4]
    # exactly as many as there are
    *got, missing = dev.pages_fork(ints(tables), ints(lens), ints(refs), ints([0, 0, -1, 0]), page)
    assert int(missing) == 0 and got[0].cpu().tolist() == [[0], [1], [-1], [2]] and got[2].cpu().tolist() == [1, 1, 1]


def test_extend_refuses_whole_or_nothing(dev):
    page = 4
    t, ln, r = ints([[0, -1], [1, 2]]), ints([3, 8]), ints([1, 1, 1, 0])
    for add, missing in (([9, 0], -1), ([0, 1], -1), ([2 ** 31 - 1, 0], -1), ([0, 0], 0), ([-5, 0], 0)):
        assert int(dev.pages_extend(t, ln, r, ints(add), page)) == missing
        assert t.cpu().tolist() == [[0, -1], [1, 2]] and ln.cpu().tolist() == [3, 8] and r.cpu().tolist() == [1, 1, 1, 0]
    t, ln, r = ints([[-1, -1], [-1, -1]]), ints([0, 0]), ints([1, 0, 1, 0, 0])
    assert int(dev.pages_extend(t, ln, r, ints([8, 8]), page)) == 1 and ln.cpu().tolist() == [0, 0] and r.cpu().tolist() == [1, 0, 1, 0, 0]
    assert int(dev.pages_extend(t, ln, r, ints([8, 4]), page)) == 0
    assert t.cpu().tolist() == [[1, 3], [4, -1]] and ln.cpu().tolist() == [8, 4] and r.cpu().tolist() == [1] * 5


def test_free(dev):
    tables, lens, refs, rng = state(40, 8, 12, 9, 10)
    tables[5, 0] = tables[6, 0] if tables[6, 0] >= 0 and tables[5, 0] >= 0 else tables[5, 0]
    refs = np.bincount(tables[tables >= 0], minlength=len(refs))
    rows = rng.rand(40) < 0.5
    t, ln, r = ints(tables), ints(lens), ints(refs)
    dev.pages_free(t, ln, r, torch.as_tensor(rows, device="cuda"), 8)
    tables[rows], lens = -1, np.where(rows, 0, lens)
    assert np.array_equal(t.cpu().numpy(), tables) and np.array_equal(ln.cpu().numpy(), lens)
    assert np.array_equal(r.cpu().numpy(), np.bincount(tables[tables >= 0], minlength=len(refs)))


@pytest.mark.parametrize("n_pages,live", [(1, 0), (1, 1), (10, 10), (10, 0), (100, 37), (1024, 512), (5000, 4999), (4096, 1500), (4097, 1), (20000, 9000), (16384, 16383), (16385, 8000), (131072, 70000)])
def test_compact(dev, n_pages, live):
    rng = np.random.RandomState(n_pages + live)
    refs = np.zeros(n_pages, np.int64)
    where = rng.permutation(n_pages)[:live]
    refs[where] = rng.randint(1, 4, live)
    tables = np.full((5, max(1, live)), -1, np.int64)
    for i in range(5):
        tables[i, : live - i * live // 7] = rng.permutation(where)[: live - i * live // 7]
    tables[4, -1] = n_pages + 5                                    # not a page: passed through
    pool = rand((3, n_pages, 2, 8), 4)
    want = pool.clone()
    remap, new_refs = np.where(refs > 0, np.arange(n_pages), -1), np.where(np.arange(n_pages) < live, refs, 0)
    src, dst = np.flatnonzero((refs > 0) & (np.arange(n_pages) >= live)), np.flatnonzero((refs == 0) & (np.arange(n_pages) < live))
    remap[src], new_refs[dst] = dst, refs[src]
    want[:, dst] = pool[:, src]
    t, r, m, s, d, count = dev.pages_compact(ints(tables), ints(refs))
    assert int(count) == len(src) == len(dst)
    assert np.array_equal(r.cpu().numpy(), new_refs) and np.array_equal(m.cpu().numpy(), remap)
    assert s[: len(src)].cpu().tolist() == src.tolist() and d[: len(src)].cpu().tolist() == dst.tolist()
    assert bool((s[len(src):] == -1).all()) and bool((d[len(src):] == -1).all())
    inside = (tables >= 0) & (tables < n_pages)
    assert np.array_equal(t.cpu().numpy(), np.where(inside, remap[np.where(inside, tables, 0)], tables))
    both = pool.clone()
    dev.pages_copy(pool, s, d, count)
    dev.pages_copy(both, s, d)
    assert torch.equal(pool, want) and torch.equal(both, want)


@pytest.mark.parametrize("shape", [(1, 5, 8), (4, 300, 16, 2, 64), (3, 20, 16, 8, 128), (2, 9, 24, 3, 72), (64, 7, 8, 1, 8), (8, 300, 16, 16, 120)])
def test_pages_copy(dev, shape):
    pool = rand(shape, 3)
    wide = torch.full((shape[0], shape[1] + 2, math.prod(shape[2:]) + 16), 5.0, dtype=torch.float16, device="cuda")     # pages apart
    view = wide[:, 1:-1, : math.prod(shape[2:])]
    view.copy_(pool.flatten(2))
    n = shape[1]
    order = np.random.RandomState(2).permutation(n)
    half = n // 2
    src, dst = order[:half], order[half: 2 * half]
    pad = np.array([-1, n, 0])
    want = pool.clone()
    want[:, dst] = pool[:, src]
    for p in (pool, view):
        dev.pages_copy(p, ints(np.concatenate([pad, src])), ints(np.concatenate([[0, 0, -1], dst])))
        assert torch.equal(p.flatten(2), want.flatten(2))
    assert bool((wide[:, 0] == 5).all()) and bool((wide[:, -1] == 5).all()) and bool((wide[..., -16:] == 5).all())
    dev.pages_copy(pool, ints(dst), ints(src), ints([0]))
    dev.pages_copy(pool, ints(dst), ints(src), ints([-3]))
    dev.pages_copy(pool, ints([]), ints([]))
    assert torch.equal(pool, want)


# ------------------------------------------------------------------------------------------------ beam search

def select(logits, scores, finished, n_beams, end, n):
    """By definition in 64 bits with a stable sort; unusable rows are at -inf."""
    x = logits.double()
    top = x.amax(-1, keepdim=True)
    base = scores.double() - (top[:, 0] + torch.log(torch.exp(x - top).sum(-1)))
    usable = torch.isfinite(base)
    s = torch.where(usable[:, None], base.nan_to_num()[:, None] + x, float("-inf"))
    s[~usable] = float("-inf")
    if finished is not None:
        stay = torch.full_like(s, float("-inf"))
        own = scores.double()
        stay[:, end] = torch.where(torch.isfinite(own), own, float("-inf"))
        s = torch.where(finished[:, None], stay, s)
    vocab = logits.shape[1]
    best, at = torch.sort(s.view(-1, n_beams * vocab), dim=1, descending=True, stable=True)
    best, at = best[:, :n], at[:, :n]
    return best.flatten(), (at % vocab).flatten().int(), (at // vocab + n_beams * torch.arange(at.shape[0], device="cuda")[:, None]).flatten().int()


def check_select(dev, logits, scores, finished, n_beams, end, n):
    want = select(logits, scores, finished, n_beams, end, n)
    got = dev.beam_select(logits, scores, n_beams, finished, end, n)
    assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
    fin = torch.isfinite(want[0])
    assert torch.equal(got[0][~fin].double(), want[0][~fin])
    off = (got[0].double() - want[0]).abs()[fin]
    assert bool((off <= 2.0 ** -24 * want[0][fin].abs() + 2.0 ** -22).all()), float(off.max())


@pytest.mark.parametrize("batch,beams,vocab,n", [(1, 1, 1, 1), (1, 4, 32000, 4), (3, 5, 32000, 10), (2, 1, 50, 50), (2, 3, 7, 21), (1, 2, 8192, 64), (5, 8, 8193, 8), (2, 4, 100003, 16),
                                                 (24, 8, 1000, 8), (22, 8, 100001, 8), (1, 40, 300, 40), (7, 3, 16385, 6), (2, 64, 257, 64), (1, 3, 2047, 3)])
def test_beam_select(dev, batch, beams, vocab, n):
    rows = batch * beams
    logits = rand((rows, vocab), 1, 2.5)
    scores = -20 * torch.rand(rows, generator=torch.Generator().manual_seed(1)).cuda()
    end = min(2, vocab - 1)
    check_select(dev, logits, scores, None, beams, end, n)
    finished = (torch.arange(rows) % 3 == 1).cuda()
    check_select(dev, logits, scores, finished, beams, end, n)
    wide = rand((rows, vocab + 5), 2)
    wide[:, 3: 3 + vocab] = logits
    check_select(dev, wide[:, 3: 3 + vocab], scores, finished, beams, end, n)


def test_beam_select_ties_go_to_the_lowest_index(dev):
    beams, vocab = 4, 20000
    rows = 2 * beams
    flat = torch.zeros((rows, vocab), dtype=torch.float16, device="cuda")
    flat[:, ::2] = -0.0                                            # the two zeros are equal
    check_select(dev, flat, torch.zeros(rows, device="cuda"), None, beams, 2, 30)
    few = (rand((rows, vocab), 3) * 2).round()                     # a handful of values, most of them many times
    few[1], few[3] = few[0], few[0]
    scores = torch.tensor([-1.0, -1.0, -2.0, -1.0] * 2, device="cuda")
    check_select(dev, few, scores, None, beams, 2, 64)
    rising = torch.linspace(-40, 40, vocab, device="cuda").half().repeat(rows, 1)       # every thread's last is its best
    check_select(dev, rising, scores, None, beams, 2, 64)
    check_select(dev, rising.flip(1).contiguous(), scores, None, beams, 2, 64)
    # a dozen low values in the right places leave a bound that thousands of logits reach
    for n in (8, 64):
        low = rand((rows, vocab), 6).abs()
        low.view(rows, -1, 8)[:, torch.arange(vocab // 8, device="cuda") % 64 < 8] -= 20
        check_select(dev, low, scores, None, beams, 2, n)
    # all beams alike, each of them with all of the answer
    same = rand((1, 5000), 7).repeat(64, 1)
    check_select(dev, same, torch.full((64,), -1.0, device="cuda"), None, 64, 2, 64)
    check_select(dev, same, -torch.arange(64, device="cuda").float() / 1024, None, 64, 2, 64)
    # a first step: all beams alike, and only the first one counts
    start = torch.tensor([0.0, -math.inf, -math.inf, -math.inf] * 2, device="cuda")
    check_select(dev, rand((1, vocab), 5).repeat(rows, 1), start, None, beams, 2, 4)


def test_beam_select_rows_without_continuations(dev):
    beams, vocab = 3, 9000
    inf, nan = math.inf, math.nan
    logits = rand((5 * beams, vocab), 4)
    logits[0] = -inf                                               # a mask that leaves nothing
    logits[1, 8999] = nan
    logits[2, 100] = inf
    logits[3:6] = -inf                                             # a request of nothing but -inf
    logits[6, 10:] = -inf                                          # a mask that leaves ten tokens
    logits[7, 1:] = -65504.0                                       # the type's lowest value as a mask
    logits[9:12] = -inf
    logits[9:12, 5:7] = 0.0                                        # six continuations in all
    scores = torch.tensor([-1.0, -2, -3, -1, -1, -1, -5, -6, -700, -1, -1, -2, -inf, nan, inf], device="cuda")
    finished = torch.zeros(15, dtype=torch.bool, device="cuda")
    for n in (1, 3, 12):
        check_select(dev, logits, scores, None, beams, 2, n)
        for rows, end in (((4,), 0), ((4, 8), 11), ((3, 4, 5, 12), 2), ((0, 1, 2, 9, 10, 11, 13, 14), 8999)):
            finished.zero_()
            finished[list(rows)] = True
            check_select(dev, logits, scores, finished, beams, end, n)


@pytest.mark.parametrize("n_in,n_out,width", [(4, 4, 16), (24, 24, 1000), (5, 9, 1), (1, 3, 257)])
def test_beam_advance(dev, n_in, n_out, width):
    rng = np.random.RandomState(width)
    history, lens = rng.randint(0, 100, (n_in, width)), rng.randint(0, width + 1, n_in)
    lens[0] = width
    finished, parents, tokens = rng.rand(n_in) < 0.3, rng.randint(0, n_in, n_out), rng.randint(0, 4, n_out)
    parents[0] = -1
    parents[-1] = n_in
    for fin in (finished, None):
        h, ln, f = dev.beam_advance(ints(history), ints(lens), None if fin is None else torch.as_tensor(fin, device="cuda"), ints(parents), ints(tokens), 2)
        for i, (p, t) in enumerate(zip(parents, tokens)):
            has = 0 <= p < n_in
            line = list(history[p][: lens[p]]) if has else []
            done = not has or (fin is not None and bool(fin[p]))
            full = not done and len(line) == width
            if not done and not full:
                line.append(t)
            assert h[i].cpu().tolist() == line + [0] * (width - len(line)) and int(ln[i]) == len(line)
            assert bool(f[i]) == (done or full or t == 2)


# ------------------------------------------------------------------------------------------------ together

def test_a_beam_search_over_the_paged_cache(dev):
    """rotary_paged, paged_attention, beam_select, beam_advance, pages_fork, pages_copy and pages_extend as a decode loop
    uses them. A token's q, k, v are a table row, so what the cache must hold follows from a beam's history alone: after
    every step each beam's pages are compared with it, and its attention with the definition."""
    requests, beams, h, kv, d, page, vocab, end = 3, 4, 8, 2, 64, 8, 500, 2
    rows, width, steps, planes = requests * beams, 8, 20, 2
    n_pages = 2 + rows * 7
    qkv = rand((vocab, (h + 2 * kv) * d), 1)
    project = rand((vocab, h * d), 2, 0.2)
    pool = torch.full((planes, n_pages, page, kv, d), float("nan"), dtype=torch.float16, device="cuda")
    kp, vp = pool[0], pool[1]
    freq = dev.rotary_frequencies(d)
    prompts = [np.random.RandomState(i).randint(3, vocab, n) for i, n in enumerate((5, 16, 23))]
    # every request's first beam holds the prompt; the others come out of the first fork
    tables, lens, refs = ints(np.full((rows, width), -1)), ints([0] * rows), ints([0] * n_pages)
    add = np.zeros(rows, np.int64)
    add[::beams] = [len(p) for p in prompts]
    assert int(dev.pages_extend(tables, lens, refs, ints(add), page)) == 0
    tokens = np.concatenate(prompts)
    seq = np.repeat(np.arange(requests) * beams, [len(p) for p in prompts])
    pos = np.concatenate([np.arange(len(p)) for p in prompts])
    x = dev.embedding(qkv, ints(tokens))
    split = lambda t: (t[:, : h * d].unflatten(1, (h, d)), t[:, h * d: (h + kv) * d].unflatten(1, (kv, d)), t[:, (h + kv) * d:].unflatten(1, (kv, d)))  # noqa: E731
    q = dev.rotary_paged(*split(x), ints(pos), ints(seq), freq, kp, vp, tables)
    last = np.cumsum([len(p) for p in prompts]) - 1
    q_rows = torch.zeros((rows, h, d), dtype=torch.float16, device="cuda")
    q_rows[::beams] = q[torch.as_tensor(last, device="cuda")]
    history, hist_lens = ints(np.zeros((rows, 64))), lens.clone()
    for i, p in enumerate(prompts):
        history[i * beams, : len(p)] = ints(p)
    scores = torch.full((rows,), -math.inf, device="cuda")
    scores[::beams] = 0.0
    finished = torch.zeros(rows, dtype=torch.bool, device="cuda")
    forked = 0
    for step in range(steps):
        out = dev.paged_attention(q_rows, kp, vp, tables, lens, 0.125, max_len=page * width)
        want, slack = attention(q_rows, kp, vp, tables.cpu().numpy(), lens.cpu().tolist(), 0.125)
        within(out, want, slack, f"step {step}")
        logits = dev.matmul2d(out.view(rows, h * d), project)
        ref = select(logits, scores, finished, beams, end, beams)
        scores, tokens, parents = dev.beam_select(logits, scores, beams, finished, end)
        assert torch.equal(tokens, ref[1]) and torch.equal(parents, ref[2])
        history, hist_lens, finished = dev.beam_advance(history, hist_lens, finished, parents, tokens, end)
        tables, lens, refs, src, dst, missing = dev.pages_fork(tables, lens, refs, parents, page)
        assert int(missing) == 0
        forked += int((src >= 0).sum())
        dev.pages_copy(pool, src, dst)
        live = (hist_lens > lens).int()                            # finished beams get no further token
        assert int(dev.pages_extend(tables, lens, refs, live, page)) == 0
        q_rows = dev.rotary_paged(*split(dev.embedding(qkv, tokens)), lens - 1, torch.where(live > 0, torch.arange(rows, device="cuda"), -1).int(), freq, kp, vp, tables)
        counted = torch.bincount(tables[tables >= 0].long(), minlength=n_pages)
        assert torch.equal(counted.int(), refs)
        for r in range(rows):
            n = int(lens[r])
            assert n == int(hist_lens[r])
            ids = history[r, :n].contiguous()
            _, k, v = split(dev.embedding(qkv, ids))
            kr = dev.rotary(k, torch.arange(n, device="cuda", dtype=torch.int32), freq)
            pages = tables[r, : -(-n // page)].long()
            assert torch.equal(kp[pages].flatten(0, 1)[:n], kr) and torch.equal(vp[pages].flatten(0, 1)[:n], v), (step, r)
        if step == steps // 2:                                     # a compaction on the way
            tables, refs, _, src, dst, count = dev.pages_compact(tables, refs)
            dev.pages_copy(pool, src, dst, count)
            assert bool((refs[: int((refs > 0).sum())] > 0).all())
    assert forked > 10
    dev.pages_free(tables, lens, refs, torch.ones(rows, dtype=torch.bool, device="cuda"), page)
    assert bool((refs == 0).all()) and bool((tables == -1).all()) and bool((lens == 0).all())


def test_a_captured_decode_step_follows_its_inputs(dev):
    """One graph of a whole step, replayed with other lengths, tables and logits; two graphs with workspaces of their own
    replayed in turn. Every replay is compared with the eager call."""
    b, h, kv, d, page, width, vocab = 4, 8, 2, 128, 16, 40, 3000
    kp, vp = paged_cache(200, page, kv, d, "row")
    freq = dev.rotary_frequencies(d)
    rng = np.random.RandomState(0)

    def inputs(seed):
        r = np.random.RandomState(seed)
        lens = r.randint(1, page * width, b)
        return dict(qkv=rand((b, (h + 2 * kv) * d), seed), lens=ints(lens), tables=ints(r.permutation(200)[: b * width].reshape(b, width)), logits=rand((b, vocab), seed + 1),
                    scores=-torch.rand(b, generator=torch.Generator().manual_seed(seed)).cuda(), refs=ints(r.randint(0, 2, 200)))

    def step(s):
        q, k, v = (s["qkv"][:, a: a + c * d].unflatten(1, (c, d)) for a, c in ((0, h), (h * d, kv), ((h + kv) * d, kv)))
        qr = dev.rotary_paged(q, k, v, s["lens"] - 1, None, freq, kp, vp, s["tables"])
        out = dev.paged_attention(qr, kp, vp, s["tables"], s["lens"], max_len=page * width)
        best = dev.beam_select(s["logits"], s["scores"], b)
        return (out, *best, *dev.pages_fork(s["tables"], s["lens"], s["refs"], best[2], page), *dev.pages_compact(s["tables"], s["refs"])[:3])

    side = torch.cuda.Stream()
    graphs = []
    try:
        for seed in (1, 2):
            s = inputs(seed)
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                dev.bind_stream(side)
                step(s)
                side.synchronize()
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=side):
                    out = step(s)
            graphs.append((g, s, out))
    finally:
        dev.bind_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    for seed in (3, 4, 5):
        for i, (g, s, _) in enumerate(graphs):
            for name, t in inputs(10 * seed + i).items():
                s[name].copy_(t)
        for g, _, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, s, out in graphs:
            k0, v0 = kp.clone(), vp.clone()
            for got, want in zip(out, step(s)):
                # both graphs wrote the shared cache before the eager steps: compare what does not depend on the order
                if got.dtype != torch.float16:
                    assert torch.equal(got, want), seed
            kp.copy_(k0), vp.copy_(v0)
        for g, s, out in graphs:                                   # alone, the whole step is the same bit for bit
            k0, v0 = kp.clone(), vp.clone()
            g.replay()
            torch.cuda.synchronize()
            got, kg, vg = [t.clone() for t in out], kp.clone(), vp.clone()
            kp.copy_(k0), vp.copy_(v0)
            want = step(s)
            assert all(torch.equal(a, c) for a, c in zip(got, want)) and torch.equal(kg, kp) and torch.equal(vg, vp)


def test_nothing_to_do(dev):
    """Empty batches, tables and pools are no error and touch nothing."""
    none, refs = torch.empty((0, 4), dtype=torch.int32, device="cuda"), ints([1, 0, 2])
    t, ln, r, src, dst, missing = dev.pages_fork(none, ints([]), refs, ints([]), 8)
    assert t.shape == (0, 4) and torch.equal(r, refs) and int(missing) == 0 and src.numel() == dst.numel() == 0
    assert int(dev.pages_extend(none, ints([]), refs, ints([]), 8)) == 0 and r.cpu().tolist() == [1, 0, 2]
    dev.pages_free(none, ints([]), refs, torch.empty(0, dtype=torch.bool, device="cuda"), 8)
    t, r, remap, src, dst, count = dev.pages_compact(none, refs)
    assert r.cpu().tolist() == [1, 2, 0] and remap.cpu().tolist() == [0, -1, 1] and int(count) == 1
    kp, vp = paged_cache(2, 8, 1, 64, "row")
    q = rand((3, 2, 64), 1)
    assert dev.paged_attention(q[:0], kp, vp, none, ints([])).shape == (0, 2, 64)
    # sequences without any table: nothing to attend to, or a length that no table covers
    got = dev.paged_attention(q, kp, vp, torch.empty((3, 0), dtype=torch.int32, device="cuda"), ints([0, 0, 1]))
    assert bool((got[:2] == 0).all()) and torch.isnan(got[2]).all()
    k0 = kp.clone()
    dev.rotary_paged(q[:0], q[:0, :1], q[:0, :1], ints([]), None, dev.rotary_frequencies(64), kp, vp, none)
    dev.rotary_paged(q, q[:, :1], q[:, :1], ints([0, 1, 2]), None, dev.rotary_frequencies(64), kp, vp, none)     # no sequence for any token
    assert torch.equal(kp, k0)
    assert all(x.numel() == 0 for x in dev.beam_select(rand((0, 10), 1), torch.empty(0, device="cuda"), 2))
    h, ln, f = dev.beam_advance(ints([[5, 6]]), ints([2]), None, ints([]), ints([]))
    assert h.shape == (0, 2) and ln.numel() == f.numel() == 0


def test_results_over_their_inputs(dev):
    """Where input and result may be the same tensor."""
    kp, vp = paged_cache(12, 8, 2, 64, "row")
    q, tables, lens = rand((3, 8, 64), 1), ints([[0, 1, 2], [3, 4, 5], [6, 7, 8]]), ints([20, 1, 9])
    want = dev.paged_attention(q, kp, vp, tables, lens)
    assert torch.equal(dev.paged_attention(q, kp, vp, tables, lens, out=q), want) and torch.equal(q, want)
    q, k, freq = rand((3, 8, 64), 1), rand((3, 2, 64), 2), dev.rotary_frequencies(64)
    want = dev.rotary_paged(q, k, k, lens, None, freq, kp, vp, tables)
    assert torch.equal(dev.rotary_paged(q, k, k, lens, None, freq, kp, vp, tables, q_out=q), want)


def test_front_end_refusals(dev):
    kv, d, page = 2, 64, 16
    kp, vp = paged_cache(4, page, kv, d, "row")
    q, k = rand((2, 4, d), 1), rand((2, kv, d), 2)
    t, ln, pos, freq = ints([[0, 1], [2, 3]]), ints([3, 4]), ints([2, 3]), dev.rotary_frequencies(d)
    for error, call in [
            (TypeError, lambda: dev.paged_attention(q.float(), kp, vp, t, ln)), (TypeError, lambda: dev.paged_attention(q, kp, vp, t.long(), ln)),
            (TypeError, lambda: dev.paged_attention(q, kp.float(), vp, t, ln)), (ValueError, lambda: dev.paged_attention(q, kp, vp[:3], t, ln)),
            (ValueError, lambda: dev.paged_attention(q, kp, vp.transpose(1, 2).contiguous().transpose(1, 2), t, ln)),
            (ValueError, lambda: dev.paged_attention(q[..., :32], kp, vp, t, ln)), (ValueError, lambda: dev.paged_attention(q, kp, vp, t[:1], ln)),
            (ValueError, lambda: dev.paged_attention(q.transpose(0, 1).contiguous().transpose(0, 1), kp, vp, t, ln)), (TensorLibError, lambda: dev.paged_attention(q.cpu(), kp, vp, t, ln)),
            (TensorLibError, lambda: dev.paged_attention(rand((2, 3, d), 1), kp, vp, t, ln)), (ValueError, lambda: dev.paged_attention(q, kp, vp, t.t(), ln)),
            (TensorLibError, lambda: dev.paged_attention(q, kp, vp, t, ln, float("nan"))),
            (TensorLibError, lambda: dev.paged_attention(q, kp, vp, t, ln, max_len=10 ** 6, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))),
            (ValueError, lambda: dev.rotary_paged(q, k[:1], k, pos, None, freq, kp, vp, t)), (ValueError, lambda: dev.rotary_paged(q, k, k, pos, None, freq, kp, vp, t, layout="both")),
            (TypeError, lambda: dev.rotary_paged(q, k, k, pos, None, freq.float(), kp, vp, t)), (ValueError, lambda: dev.rotary_paged(q, k, k, pos[:1], None, freq, kp, vp, t)),
            (TensorLibError, lambda: dev.rotary(q, pos, dev.rotary_frequencies(128))), (ValueError, lambda: dev.rotary_frequencies(64, scaling="cubic")),
            (ValueError, lambda: dev.pages_fork(t, ln, ints([1] * 4), ints([0]), page)), (TensorLibError, lambda: dev.pages_fork(t, ln, ints([1] * 4), ints([0, 1]), 0)),
            (ValueError, lambda: dev.pages_copy(torch.empty(2, 4, 8, 8, dtype=torch.float16, device="cuda").transpose(2, 3), ints([0]), ints([1]))),
            (TensorLibError, lambda: dev.pages_copy(torch.empty(2, 4, 3, dtype=torch.float16, device="cuda"), ints([0]), ints([1]))),
            (TypeError, lambda: dev.pages_free(t, ln, ints([1] * 4), ints([0, 1]), page)),
            (ValueError, lambda: dev.beam_select(rand((5, 10), 1), torch.zeros(5, device="cuda"), 2)), (TensorLibError, lambda: dev.beam_select(rand((4, 10), 1), torch.zeros(4, device="cuda"), 2, n_select=65)),
            (TypeError, lambda: dev.beam_select(rand((4, 10), 1), torch.zeros(4, device="cuda").double(), 2)),
            (ValueError, lambda: dev.beam_advance(ints([[1, 2]]), ints([1]), None, ints([0, 0]), ints([1])))]:
        with pytest.raises(error):
            call()
    with torch.cuda.stream(torch.cuda.Stream()):                   # not the stream the library enqueues on
        with pytest.raises(TensorLibError, match="stream"):
            dev.paged_attention(q, kp, vp, t, ln)


def test_results_are_the_callers_own(dev):
    """Results that share an allocation: apart from each other, usable on their own, alive when the others are gone, and
    not written by later calls."""
    for rows, width, pages in ((3, 5, 70), (1, 1, 1), (65, 63, 4096)):
        tables = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")
        lens = torch.zeros(rows, dtype=torch.int32, device="cuda")
        refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
        parents = torch.arange(rows, dtype=torch.int32, device="cuda")
        first = dev.pages_fork(tables, lens, refs, parents, 4)
        spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in first)
        assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:]))
        assert all(t.is_contiguous() and not t.requires_grad and t.is_leaf and t._version == 0 for t in first)
        for i, t in enumerate(first):
            t.fill_(100 + i)
        second = dev.pages_fork(tables, lens, refs, parents, 4)
        assert all(bool((t == 100 + i).all()) for i, t in enumerate(first))
        kept = second[2]
        del second
        other = [torch.full((pages,), 7, dtype=torch.int32, device="cuda") for _ in range(8)]
        assert not kept.any() and all(bool((t == 7).all()) for t in other)
    with torch.inference_mode():
        history = torch.zeros((4, 8), dtype=torch.int32, device="cuda")
        lens = torch.zeros(4, dtype=torch.int32, device="cuda")
        ids = torch.arange(4, dtype=torch.int32, device="cuda")
        h2, l2, f2 = dev.beam_advance(history, lens, None, ids, ids + 5, end_token=6)
        assert h2.is_inference() and h2[:, 0].tolist() == [5, 6, 7, 8] and l2.tolist() == [1] * 4
        assert f2.dtype == torch.bool and f2.tolist() == [False, True, False, False]
    h2, l2, f2 = dev.beam_advance(history, lens, f2, ids, ids, end_token=6)
    assert f2.logical_not().tolist() == [True, False, True, True]


def test_calls_from_several_threads(dev):
    """The library's errors are per thread and a launch runs without the interpreter's lock."""
    import threading
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn((40, 4, 64), generator=g, device="cuda", dtype=torch.float16)
    positions = torch.arange(40, dtype=torch.int32, device="cuda")
    freq = dev.rotary_frequencies(64)
    want = dev.rotary(x, positions, freq)
    wrong = []

    def right():
        for _ in range(50):
            if not torch.equal(dev.rotary(x, positions, freq), want):
                wrong.append("result")

    def refused():
        for _ in range(50):
            try:
                dev.rotary(x[..., :63].contiguous(), positions, freq)
                wrong.append("no refusal")
            except TensorLibError as e:
                if "tl_rotary_f16" not in str(e):
                    wrong.append(str(e))

    threads = [threading.Thread(target=t) for t in (right, refused, right)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[:3]


def test_the_current_device_and_stream_are_checked(dev):
    """What allocates runs on torch's current stream only; what does not may run on the library's own."""
    pool = rand((2, 6, 16), 1)
    want = pool.clone()
    want[:, 3] = pool[:, 5]
    tables, lens, refs = ints([[0, 1]]), ints([7]), ints([1, 1, 0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    dev.bind_stream(side)
    try:
        for call in (lambda: dev.pages_extend(tables, lens, refs, ints([1]), 4), lambda: dev.rotary(rand((1, 1, 8), 2), ints([0]), dev.rotary_frequencies(8))):
            with pytest.raises(TensorLibError, match="stream"):
                call()
        dev.pages_copy(pool, ints([5]), ints([3]))
        torch.cuda.synchronize()
        assert torch.equal(pool, want) and lens.tolist() == [7]
    finally:
        dev.bind_stream(torch.cuda.current_stream())


@pytest.mark.parametrize("n", [1, 8, 9, 64])
def test_beam_select_when_the_bound_is_loose(dev, n):
    """A quarter of each slice low, so that its wavefront's share is no bound for the rest; masks that leave fewer tokens than are
    selected; slices of every length at the end."""
    beams = 3
    scores = torch.tensor([-1.0, -1.5, -1.25], device="cuda")
    for vocab in (8192 * 86, 20000):                               # both slice lengths
        for part in range(4):
            low = rand((beams, vocab), 6 + part).abs()
            low.view(beams, -1, 8)[:, torch.arange(vocab // 8, device="cuda") % 256 // 64 == part] -= 20
            check_select(dev, low, scores, None, beams, 2, n)
    for vocab in (2049, 2048 + 511, 2048 + 1791, 2048 + 1792, 4095, 4096):
        masked = torch.full((beams, vocab), -math.inf, dtype=torch.float16, device="cuda")
        masked[:, torch.randperm(vocab, generator=torch.Generator().manual_seed(vocab))[:5].cuda()] = rand((beams, 5), 3)
        check_select(dev, masked, scores, None, beams, 2, n)
        check_select(dev, rand((beams, vocab), 4), scores, None, beams, 2, n)


# ------------------------------------------------------------------------------------------------ long lists of the pick

def select_into(dev, logits, scores, finished, n_beams, end, n):
    """tl_beam_select_f16 itself, with outputs that hold something beforehand: a place that is not written shows."""
    import ctypes
    rows, vocab = logits.shape
    batch = rows // n_beams
    out = (torch.full((batch * n,), 12345.0, device="cuda"), ints([-77] * (batch * n)), ints([-99] * (batch * n)))
    ws = torch.empty(dev.beam_select_workspace(batch, n_beams, vocab, n), dtype=torch.uint8, device="cuda")
    p = lambda t: None if t is None else ctypes.c_void_p(t.data_ptr())  # noqa: E731
    rc = dev.lib.tl_beam_select_f16(p(out[0]), p(out[1]), p(out[2]), p(logits), logits.stride(0), p(scores), p(finished), batch, n_beams, vocab, n, end, p(ws), ws.numel())
    assert rc == 0, dev.lib.tl_last_error()
    return out


def check_select_into(dev, logits, scores, finished, n_beams, end, n):
    """Tolerance of a score: half an fp32 step, and the logarithm of a row's sum, whose exponentials are good to an ulp (2^-23) and
    whose additions within a thread are fp32, eight roundings in turn (8 * 2^-24): below 2^-20 together."""
    want = select(logits, scores, finished, n_beams, end, n)
    got = select_into(dev, logits, scores, finished, n_beams, end, n)
    assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
    fin = torch.isfinite(want[0])
    assert torch.equal(got[0][~fin].double(), want[0][~fin])
    off = (got[0].double() - want[0]).abs()[fin]
    assert bool((off <= 2.0 ** -24 * want[0][fin].abs() + 2.0 ** -20).all()), float(off.max())


@pytest.mark.parametrize("batch,beams,vocab,n,allowed", [(1, 4, 128256, 4, (100, 60000)), (1, 4, 50257, 8, (7, 50256)), (1, 8, 32000, 8, (31999,)), (1, 4, 100003, 4, (0, 99999)),
                                                         (24, 8, 100003, 8, (70001,)), (3, 5, 32000, 10, (2, 16000, 31000))])
def test_beam_select_under_a_mask_that_leaves_a_few_tokens(dev, batch, beams, vocab, n, allowed):
    """Constrained decoding: all but a few tokens at -inf, the same ones in every beam. Most candidates are at -inf, too many
    threads have nothing better for a bound, and hundreds of candidates are ranked; the best beam is the last one."""
    rows = batch * beams
    logits = torch.full((rows, vocab), -math.inf, dtype=torch.float16, device="cuda")
    logits[:, list(allowed)] = rand((rows, len(allowed)), 5)
    finished = (torch.arange(rows) % 3 == 1).cuda()
    for scores in (torch.arange(rows, device="cuda") / 4.0 - 60.0, -torch.arange(rows, device="cuda") / 4.0):
        check_select_into(dev, logits, scores, None, beams, 2, n)
        check_select_into(dev, logits, scores, finished, beams, 2, n)


@pytest.mark.parametrize("beams,slices,n,rest", [(8, 8, 8, 2048), (3, 9, 19, 19), (8, 16, 8, 8), (3, 11, 31, 2047), (5, 5, 41, 100), (7, 11, 13, 300), (1, 16, 64, 64), (8, 10, 8, 9), (1, 8, 64, 64),
                                                  (1, 17, 61, 61)])
@pytest.mark.parametrize("step", [0.0, 2.0 ** -20, -2.0 ** -20])
def test_beam_select_of_lists_of_any_length(dev, beams, slices, n, rest, step):
    """Rows of equal logits: every candidate reaches the bound, so the list is as long as there are candidates (beams x slices x
    n: 512, 513, 1024, 1023, 1025, 1001, 1024, 640, 512, 1037), whether the beams are equal, the last one the best or the first."""
    vocab = (slices - 1) * 2048 + rest
    logits = torch.full((beams, vocab), 1.5, dtype=torch.float16, device="cuda")
    scores = -1.0 + step * torch.arange(beams, device="cuda", dtype=torch.float32)
    check_select_into(dev, logits, scores, None, beams, 2, n)


def test_one_workspace_for_every_bound_and_batch(dev):
    """A workspace sized once for the limit of a program serves its shorter bounds and smaller batches."""
    h, kv, d, page, lens = 32, 8, 128, 16, [20000, 700, 4097]
    tables, n_pages = tables_for(lens, page)
    kp, vp = paged_cache(n_pages, page, kv, d, "row")
    q = rand((3, h, d), 8)
    ws = torch.empty(dev.paged_attention_workspace(3, h, kv, d, 131072), dtype=torch.uint8, device="cuda")
    for rows in (slice(0, 3), slice(0, 1), slice(1, 3), slice(1, 2)):
        for bound in (20000, 25000, 73728, 131072):
            args = q[rows], kp, vp, ints(tables[rows]), ints(lens[rows])
            ws.fill_(255)                                          # NaN, whatever is read of it
            assert torch.equal(dev.paged_attention(*args, max_len=bound, workspace=ws), dev.paged_attention(*args, max_len=bound)), (rows, bound)


def test_one_workspace_for_every_beam_batch(dev):
    """A workspace sized once for the largest batch serves the smaller ones, whose rows are cut more finely."""
    beams, vocab, most = 4, 100003, 12
    logits, scores = rand((most * beams, vocab), 3, 2.5), -20 * torch.rand(most * beams, generator=torch.Generator().manual_seed(1)).cuda()
    ws = torch.empty(dev.beam_select_workspace(most, beams, vocab, beams), dtype=torch.uint8, device="cuda")
    for batch in (most, 5, 4, 2, 1):
        ws.fill_(255)
        args = logits[: batch * beams], scores[: batch * beams], beams
        assert all(torch.equal(a, b) for a, b in zip(dev.beam_select(*args, workspace=ws), dev.beam_select(*args)))


def test_calls_on_another_stream_than_torchs_stay_in_line(dev):
    """pages_copy and pages_free may run on a library stream that is not torch's current one: behind what made their tensors
    there, ahead of what reads them and of what has their memory next."""
    pool, wait = rand((4, 60, 8, 64), 1), 20_000_000               # cycles, some ten milliseconds
    src, dst = np.arange(0, 30), np.arange(59, 29, -1)
    want = pool.clone()
    want[:, dst] = pool[:, src]
    tables, lens, refs, _ = state(40, 8, 12, 9, 10)
    rows = np.arange(40) % 3 == 0
    left = np.where(rows[:, None], -1, tables)
    device_src, device_dst = ints(src), ints(dst)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    dev.bind_stream(side)
    try:
        for slow in (torch.cuda.current_stream(), side):
            p, t, ln, r = torch.zeros_like(pool), ints(np.full_like(tables, -1)), ints(np.zeros_like(lens)), ints(np.zeros_like(refs))
            values = [pool, ints(tables), ints(lens), ints(refs)]
            torch.cuda.synchronize()
            with torch.cuda.stream(slow):
                torch.cuda._sleep(wait)
            for to, x in zip((p, t, ln, r), values):
                to.copy_(x)                                        # the operands are there only now
            ids = device_src + 0, device_dst + 0
            dev.pages_copy(p, *ids)
            del ids
            other = torch.full((30,), 7, dtype=torch.int32, device="cuda"), torch.full((30,), 7, dtype=torch.int32, device="cuda")
            which = torch.as_tensor(rows, device="cuda")
            dev.pages_free(t, ln, r, which, 8)
            which.zero_()                                          # and its readers wait
            got = [x.clone() for x in (p, t, ln, r)]
            torch.cuda.synchronize()
            assert torch.equal(got[0], want) and all(bool((o == 7).all()) for o in other)
            assert np.array_equal(got[1].cpu().numpy(), left) and np.array_equal(got[2].cpu().numpy(), np.where(rows, 0, lens))
            assert np.array_equal(got[3].cpu().numpy(), np.bincount(left[left >= 0], minlength=len(refs)))
    finally:
        dev.bind_stream(torch.cuda.current_stream())


def test_captures_and_another_library_stream(dev):
    """A capture of torch's stream would go without a call that the library enqueues elsewhere: refused, and the capture goes on.
    A capture of the library's own stream records it, whatever torch's current stream is."""
    pool, src, dst = rand((2, 6, 16), 1), ints([5, 1]), ints([3, 0])
    kept, want = pool.clone(), pool.clone()
    want[:, [3, 0]] = pool[:, [5, 1]]
    state_ = ints([[0, 1]]), ints([7]), ints([1, 1, 0]), torch.ones(1, dtype=torch.bool, device="cuda")
    side, main = torch.cuda.Stream(), torch.cuda.current_stream()
    x = torch.zeros(8, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        for call in (lambda: dev.pages_copy(pool, src, dst), lambda: dev.pages_free(*state_, 4)):
            with pytest.raises(TensorLibError, match="captured"):
                call()
        x += 1
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(pool, kept) and bool((x == 1).all()) and state_[1].tolist() == [7]
    g = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(g, stream=side):
            dev.bind_stream(side)
            with torch.cuda.stream(main):
                dev.pages_copy(pool, src, dst)
    finally:
        dev.bind_stream(main)
    for _ in range(3):
        pool.copy_(kept)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(pool, want)


def test_a_captured_beam_step_with_its_pages(dev):
    """Selection, histories, fork, copy, extension and release of finished rows in one graph, what works in place included:
    replayed with other inputs, eager work between the replays, each compared with the eager step and with the plain loops."""
    requests, beams, page, width, vocab, planes, history = 5, 4, 8, 6, 3000, 3, 60
    rows = requests * beams
    n_pages = rows * width + 40

    def inputs(seed):
        r = np.random.RandomState(seed)
        tables, lens, refs, _ = state(rows, page, width, seed, 40, r.randint(1, page * width - 1, rows))
        refs = np.concatenate([refs, np.zeros(n_pages - len(refs), int)])
        return dict(logits=rand((rows, vocab), seed, 2.5), scores=-torch.rand(rows, generator=torch.Generator().manual_seed(seed)).cuda(), finished=torch.as_tensor(r.rand(rows) < 0.2, device="cuda"),
                    history=ints(r.randint(0, vocab, (rows, history))), hist_lens=ints(r.randint(1, history, rows)), tables=ints(tables), lens=ints(lens), refs=ints(refs),
                    pool=rand((planes, n_pages, page, 2, 8), seed + 1))

    def step(s):
        scores, tokens, parents = dev.beam_select(s["logits"], s["scores"], beams, s["finished"], 2)
        hist, hist_lens, finished = dev.beam_advance(s["history"], s["hist_lens"], s["finished"], parents, tokens, 2)
        tables, lens, refs, src, dst, lacking = dev.pages_fork(s["tables"], s["lens"], s["refs"], parents, page)
        dev.pages_copy(s["pool"], src, dst)
        short = dev.pages_extend(tables, lens, refs, finished.logical_not().int(), page)
        forked = tables.clone(), lens.clone(), refs.clone()
        dev.pages_free(tables, lens, refs, finished, page)
        return scores, tokens, parents, hist, hist_lens, finished, src, dst, lacking, short, *forked, tables, lens, refs

    side, s = torch.cuda.Stream(), inputs(1)
    torch.cuda.synchronize()
    try:
        with torch.cuda.stream(side):
            dev.bind_stream(side)
            step(s)
            side.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                out = step(s)
    finally:
        dev.bind_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    for seed in (2, 3, 4, 5):
        fresh = inputs(seed)
        for name, t in fresh.items():
            s[name].copy_(t)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = step(fresh)                                         # eager, on inputs of its own
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(s["pool"], fresh["pool"]), seed
        start = inputs(seed)
        tables, lens, refs, src, dst = fork_by_hand(*(start[k].cpu().numpy() for k in ("tables", "lens", "refs")), got[2].cpu().tolist(), page)
        assert got[6].cpu().tolist() == src and got[7].cpu().tolist() == dst and int(got[8]) == int(got[9]) == 0
        pool = start["pool"]
        for a, b in zip(src, dst):
            if a >= 0:
                pool[:, b] = pool[:, a]
        assert torch.equal(s["pool"], pool)
        done = got[5].cpu().tolist()
        for i in range(rows):
            if not done[i] and lens[i] % page == 0:
                tables[i][lens[i] // page] = refs.index(0)
                refs[refs.index(0)] = 1
            lens[i] += not done[i]
        assert [t.cpu().tolist() for t in got[10:13]] == [tables, lens, refs]
        for i in range(rows):
            if done[i]:
                for p in tables[i][: -(-lens[i] // page)]:
                    refs[p] -= 1
                tables[i], lens[i] = [-1] * width, 0
        assert [t.cpu().tolist() for t in got[13:]] == [tables, lens, refs]


@pytest.mark.parametrize("batch,beams,vocab,n,masked", [(1, 8, 1, 8, -math.inf), (3, 4, 32000, 4, -math.inf), (2, 8, 100003, 8, -65504.0), (9, 8, 50257, 8, -math.inf), (1, 64, 5000, 64, -math.inf),
                                                        (1, 3, 600001, 2, -65504.0)])
def test_beam_select_of_one_allowed_token(dev, batch, beams, vocab, n, masked):
    """A row with one token left continues with probability 1: its score stays what it was, to the bit, and beams of equal scores
    come in their order, whatever the token's logit is and wherever it stands."""
    rows = batch * beams
    rng = np.random.RandomState(vocab)
    logits = torch.full((rows, vocab), masked, dtype=torch.float16, device="cuda")
    token = torch.as_tensor(rng.randint(0, vocab, rows), device="cuda")
    logits[torch.arange(rows, device="cuda"), token] = rand((rows,), 9, 8.0)
    for scores in (torch.zeros(rows, device="cuda"), torch.full((rows,), -3.1875, device="cuda"), torch.as_tensor(-rng.randint(0, 3, rows) - 0.3, dtype=torch.float32, device="cuda"),
                   -20 * torch.rand(rows, generator=torch.Generator().manual_seed(1)).cuda()):
        got = select_into(dev, logits, scores, None, beams, 0, n)
        order = torch.sort(scores.view(batch, beams), dim=1, descending=True, stable=True)
        parents = (order.indices[:, :n] + beams * torch.arange(batch, device="cuda")[:, None]).flatten()
        assert torch.equal(got[2], parents.int()) and torch.equal(got[1], token[parents].int())
        assert torch.equal(got[0], scores[parents])
