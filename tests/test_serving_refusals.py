"""What the serving entry points (rotary, paged attention, page bookkeeping, beam search) refuse, and the rotary
frequencies: host code, no GPU. The C entry points check every argument before they touch the device, so calls with
made-up pointers come back with TL_EINVAL / TL_ELIMIT and a message."""
import ctypes
import math
import re

import numpy as np
import pytest

from tensorlib_amd import _lib
from tensorlib_amd._lib import KvPages

TL_EINVAL, TL_ELIMIT = -1, -4
P = 0x1000          # an aligned pointer that is never followed
F32 = ctypes.c_float


def call(name, *args):
    lib = _lib.lib()
    rc = getattr(lib, name)(*args)
    return rc, lib.tl_last_error().decode()


def refused(name, args, match, code=TL_EINVAL):
    rc, msg = call(name, *args)
    assert rc == code, (rc, msg)
    assert match in msg, msg


def changed(good, **kw):
    d = dict(good)
    d.update(kw)
    return list(d.values())


def cache(**kw):
    d = dict(k=P, v=P, page_stride=16 * 2 * 64, row_stride=2 * 64, head_stride=64, n_pages=4, page_size=16, n_kv_heads=2, head_dim=64)
    d.update(kw)
    return KvPages(*d.values())


ROTARY = dict(out=P, out_stride=128, x=P, in_stride=128, positions=P, freq=P, rotary_dim=32, layout=1, magnitude=1.0, n_tokens=3, n_heads=2, head_dim=64)
ROTARY_PAGED = dict(q_out=P, q=P, q_stride=512, k=P, k_stride=512, v=P, v_stride=512, positions=P, seq_ids=None, freq=P, rotary_dim=64, layout=0,
                    magnitude=1.0, n_tokens=3, n_heads=4, cache=None, tables=P, table_stride=4, n_seqs=3)
ATTENTION = dict(out=P, q=P, q_stride=256, cache=None, tables=P, table_stride=4, lens=P, n_seqs=3, n_heads=4, max_len=64, scale=0.125, ws=None, ws_bytes=0)
FORK = dict(tables=P, lens=P, refs=P, parents=P, tables_out=2 * P, lens_out=2 * P, refs_out=2 * P, src=P, dst=P, missing=P, n_seqs=4, table_stride=8,
            n_pages=16, page_size=16)
EXTEND = dict(tables=P, lens=P, refs=P, add=P, missing=P, n_seqs=4, table_stride=8, n_pages=16, page_size=16)
FREE = dict(tables=P, lens=P, refs=P, rows=P, n_seqs=4, table_stride=8, n_pages=16, page_size=16)
COMPACT = dict(tables=P, refs=P, tables_out=P, refs_out=2 * P, remap=P, src=P, dst=P, count=P, n_seqs=4, table_stride=8, n_pages=16)
COPY = dict(pool=P, plane_stride=4096, page_stride=256, page_bytes=256, n_planes=2, n_pages=16, src=P, dst=P, count=None, max_pairs=4)
SELECT = dict(scores_out=P, tokens_out=P, parents_out=P, logits=P, logits_stride=100, scores=P, finished=None, n_batch=2, n_beams=4, vocab=100, n_select=4,
              end_token=2, ws=P, ws_bytes=1 << 20)
ADVANCE = dict(history_out=P, lens_out=P, finished_out=P, history=2 * P, lens=2 * P, finished=None, parents=P, tokens=P, n_in=4, n_out=4, stride=8, end=2)


@pytest.mark.parametrize("kw,match", [
    (dict(rotary_dim=33), "rotary_dim"), (dict(rotary_dim=66), "rotary_dim"), (dict(rotary_dim=-2), "rotary_dim"), (dict(layout=2), "layout"),
    (dict(magnitude=math.nan), "magnitude"), (dict(magnitude=math.inf), "magnitude"), (dict(n_tokens=-1), "negative"), (dict(n_heads=-1), "negative"),
    (dict(positions=None), "null"), (dict(freq=None), "null"), (dict(x=None), "null"), (dict(out=None), "null"), (dict(in_stride=127), "stride"),
    (dict(out_stride=127), "stride"), (dict(out_stride=256), "in place"), (dict(head_dim=0), "rotary_dim")])
def test_rotary_refuses(kw, match):
    refused("tl_rotary_f16", changed(ROTARY, **kw), match)


def test_sizes_past_a_launch_are_refused():
    many = dict(n_tokens=1 << 20, n_heads=1 << 12, in_stride=1 << 18, out_stride=1 << 18)
    refused("tl_rotary_f16", changed(ROTARY, **many), "too many", TL_ELIMIT)
    refused("tl_rotary_f16", changed(ROTARY, n_tokens=1, n_heads=2 ** 31 - 1), "too many", TL_ELIMIT)
    refused("tl_rotary_kv_pages_f16", changed(ROTARY_PAGED, n_tokens=1, n_heads=1, rotary_dim=0, cache=cache(n_kv_heads=2 ** 31 - 1, head_dim=8)), "too many",
            TL_ELIMIT)
    args = changed(ATTENTION, cache=cache(), n_seqs=65535, max_len=200000, ws=P, ws_bytes=1 << 40)
    refused("tl_paged_attention_f16", args, "too many", TL_ELIMIT)


def test_rotary_of_no_tokens():
    rc, _ = call("tl_rotary_f16", *changed(ROTARY, n_tokens=0, out=None, x=None, positions=None, freq=None))
    assert rc == 0          # nothing to do is no error


@pytest.mark.parametrize("kw,match", [
    (dict(k=None), "null"), (dict(v=None), "null"), (dict(tables=None), "null"), (dict(q=None), "null"), (dict(q_out=None), "null"),
    (dict(positions=None), "null"), (dict(q_stride=255), "stride"), (dict(k_stride=127), "stride"), (dict(v_stride=127), "stride"),
    (dict(rotary_dim=66), "rotary_dim"), (dict(n_seqs=-1), "negative"), (dict(layout=-1), "layout")])
def test_rotary_paged_refuses(kw, match):
    args = dict(ROTARY_PAGED, cache=cache())
    refused("tl_rotary_kv_pages_f16", changed(args, **kw), match)


BAD_CACHES = [(dict(k=None), "null"), (dict(v=None), "null"), (dict(n_pages=0), "positive"), (dict(page_size=0), "positive"), (dict(n_kv_heads=0), "positive"),
              (dict(head_dim=12), "head_dim"), (dict(head_dim=264), "head_dim"), (dict(head_dim=0), "head_dim"), (dict(k=P + 2), "aligned"),
              (dict(v=P + 8), "aligned"), (dict(page_stride=100), "strides"), (dict(row_stride=12), "strides"), (dict(head_stride=4), "strides")]


@pytest.mark.parametrize("kw,match", BAD_CACHES)
def test_bad_cache_descriptions(kw, match):
    refused("tl_rotary_kv_pages_f16", changed(ROTARY_PAGED, cache=cache(**kw)), match)
    refused("tl_paged_attention_f16", changed(ATTENTION, cache=cache(**kw)), match)


@pytest.mark.parametrize("kw,match", [
    (dict(n_heads=3), "share"), (dict(n_heads=0), "out of range"), (dict(n_seqs=-1), "out of range"), (dict(max_len=-1), "out of range"),
    (dict(scale=math.nan), "scale"), (dict(out=None), "null"), (dict(q=None), "null"), (dict(lens=None), "null"), (dict(tables=None), "null"),
    (dict(q=P + 2), "aligned"), (dict(q_stride=260), "aligned"), (dict(q_stride=248), "stride"),
    (dict(max_len=100000), "workspace"), (dict(max_len=100000, ws=P, ws_bytes=1000), "workspace"), (dict(max_len=100000, ws=P + 4, ws_bytes=1 << 30), "workspace")])
def test_attention_refuses(kw, match):
    args = dict(ATTENTION, cache=cache())
    refused("tl_paged_attention_f16", changed(args, **kw), match)


def test_attention_limits_and_empty_batch():
    args = dict(ATTENTION, cache=cache())
    refused("tl_paged_attention_f16", changed(args, n_seqs=65536, q_stride=256, ws=P, ws_bytes=1 << 40), "too many", TL_ELIMIT)
    assert call("tl_paged_attention_f16", *changed(args, n_seqs=0, out=None, q=None, lens=None, tables=None))[0] == 0
    lib = _lib.lib()
    assert lib.tl_paged_attention_workspace(0, 4, 2, 64, 100) == 0
    assert lib.tl_paged_attention_workspace(4, 4, 3, 64, 100) == 0
    need = lib.tl_paged_attention_workspace(4, 4, 2, 64, 100000)
    assert need > 0 and need % ((64 + 2) * 4 * 4 * 4) == 0


@pytest.mark.parametrize("name,good,kw,match,code", [
    ("tl_pages_fork", FORK, dict(refs=None), "null", TL_EINVAL), ("tl_pages_fork", FORK, dict(parents=None), "null", TL_EINVAL),
    ("tl_pages_fork", FORK, dict(src=None), "null", TL_EINVAL), ("tl_pages_fork", FORK, dict(tables_out=P), "over the old", TL_EINVAL),
    ("tl_pages_fork", FORK, dict(refs_out=P), "over the old", TL_EINVAL), ("tl_pages_fork", FORK, dict(lens_out=P), "over the old", TL_EINVAL),
    ("tl_pages_fork", FORK, dict(n_seqs=8193), "at most", TL_ELIMIT), ("tl_pages_fork", FORK, dict(page_size=0), "out of range", TL_EINVAL),
    ("tl_pages_fork", FORK, dict(n_seqs=8192, table_stride=1 << 20), "too large", TL_ELIMIT),
    ("tl_pages_extend", EXTEND, dict(add=None), "null", TL_EINVAL), ("tl_pages_extend", EXTEND, dict(missing=None), "null", TL_EINVAL),
    ("tl_pages_extend", EXTEND, dict(n_seqs=-1), "out of range", TL_EINVAL), ("tl_pages_extend", EXTEND, dict(table_stride=0), "out of range", TL_EINVAL),
    ("tl_pages_free", FREE, dict(rows=None), "null", TL_EINVAL), ("tl_pages_free", FREE, dict(n_pages=0), "out of range", TL_EINVAL),
    ("tl_pages_compact", COMPACT, dict(remap=None), "null", TL_EINVAL), ("tl_pages_compact", COMPACT, dict(refs_out=P), "over the old", TL_EINVAL),
    ("tl_pages_compact", COMPACT, dict(n_pages=0), "out of range", TL_EINVAL), ("tl_pages_compact", COMPACT, dict(tables=None), "null", TL_EINVAL),
    ("tl_pages_copy", COPY, dict(pool=None), "null", TL_EINVAL), ("tl_pages_copy", COPY, dict(src=None), "null", TL_EINVAL),
    ("tl_pages_copy", COPY, dict(page_bytes=250), "16 bytes", TL_EINVAL), ("tl_pages_copy", COPY, dict(pool=P + 8), "16 bytes", TL_EINVAL),
    ("tl_pages_copy", COPY, dict(plane_stride=4100), "16 bytes", TL_EINVAL), ("tl_pages_copy", COPY, dict(page_stride=128), "overlap", TL_EINVAL),
    ("tl_pages_copy", COPY, dict(max_pairs=-1), "negative", TL_EINVAL),
    ("tl_pages_copy", COPY, dict(page_bytes=1 << 40, page_stride=1 << 40), "too much", TL_ELIMIT),
    ("tl_beam_select_f16", SELECT, dict(logits=None), "null", TL_EINVAL), ("tl_beam_select_f16", SELECT, dict(scores=None), "null", TL_EINVAL),
    ("tl_beam_select_f16", SELECT, dict(n_select=65), "at most", TL_ELIMIT), ("tl_beam_select_f16", SELECT, dict(n_beams=1025), "at most", TL_ELIMIT),
    ("tl_beam_select_f16", SELECT, dict(n_beams=1, vocab=3), "do not exist", TL_EINVAL), ("tl_beam_select_f16", SELECT, dict(finished=P, end_token=100), "outside", TL_EINVAL),
    ("tl_beam_select_f16", SELECT, dict(finished=P, end_token=-1), "outside", TL_EINVAL), ("tl_beam_select_f16", SELECT, dict(logits_stride=99), "stride", TL_EINVAL),
    ("tl_beam_select_f16", SELECT, dict(ws_bytes=10), "workspace", TL_EINVAL), ("tl_beam_select_f16", SELECT, dict(ws=None), "workspace", TL_EINVAL),
    ("tl_beam_select_f16", SELECT, dict(logits=P + 1), "misaligned", TL_EINVAL), ("tl_beam_select_f16", SELECT, dict(n_batch=20000, ws_bytes=1 << 40), "at most", TL_ELIMIT),
    ("tl_beam_advance", ADVANCE, dict(parents=None), "null", TL_EINVAL), ("tl_beam_advance", ADVANCE, dict(history_out=2 * P), "over the old", TL_EINVAL),
    ("tl_beam_advance", ADVANCE, dict(n_out=65536), "at most", TL_ELIMIT), ("tl_beam_advance", ADVANCE, dict(stride=0), "out of range", TL_EINVAL)])
def test_pages_and_beam_refuse(name, good, kw, match, code):
    refused(name, changed(good, **kw), match, code)


def frequencies(rotary_dim, base=10000.0, scaling=0, factor=1.0, context=0.0, slow=1.0, fast=32.0):
    out = np.full(max(rotary_dim // 2, 1), np.nan)
    rc, msg = call("tl_rotary_frequencies", out.ctypes.data_as(ctypes.c_void_p), rotary_dim, base, scaling, factor, context, slow, fast)
    return rc, msg, out


@pytest.mark.parametrize("rd", [2, 4, 20, 64, 128, 256])
@pytest.mark.parametrize("base", [10000.0, 500000.0])
def test_frequencies_follow_the_formulas(rd, base):
    # pow is accurate to about an ulp, and a handful of operations follow: 16 * 2^-53
    tol = dict(rtol=16 * 2.0 ** -53, atol=0)
    i = np.arange(rd // 2, dtype=np.float64)
    f = base ** (-2 * i / rd)
    assert np.allclose(frequencies(rd, base)[2], f, **tol)
    assert np.allclose(frequencies(rd, base, 1, 8.0)[2], f / 8, **tol)
    if rd > 2:
        # the exponent -2 i / rd is up to 1 and multiplies the logarithm of the base: its rounding moves the power by ln(base) * 2^-53
        g = frequencies(rd, base, 2, 8.0)[2]
        assert np.allclose(g, (base * 8.0 ** (rd / (rd - 2))) ** (-2 * i / rd), rtol=64 * 2.0 ** -53, atol=0)
        assert math.isclose(g[-1], f[-1] / 8, rel_tol=64 * 2.0 ** -53)      # the last pair slows down by the factor
    g = frequencies(rd, base, 3, 8.0, 4096.0, 1.0, 32.0)[2]
    turns = 4096.0 * f / (2 * math.pi)
    keep = np.clip((turns - 1) / 31, 0, 1)
    # where turns is close to `slow` the difference cancels: turns carries 3 roundings of up to 32, divided by 31
    assert np.allclose(g, f * keep + f / 8 * (1 - keep), rtol=64 * 2.0 ** -53, atol=0)
    assert np.all(g[turns >= 32] == f[turns >= 32]) or np.allclose(g[turns >= 32], f[turns >= 32], **tol)


@pytest.mark.parametrize("args,match", [
    (dict(rotary_dim=0), "even"), (dict(rotary_dim=7), "even"), (dict(rotary_dim=8, base=0.0), "base"), (dict(rotary_dim=8, base=math.inf), "base"),
    (dict(rotary_dim=8, scaling=4), "scaling"), (dict(rotary_dim=8, scaling=1, factor=0.0), "factor"), (dict(rotary_dim=2, scaling=2, factor=2.0), "rotary_dim"),
    (dict(rotary_dim=8, scaling=3, factor=2.0), "original_context"), (dict(rotary_dim=8, scaling=3, factor=2.0, context=10.0, slow=4.0, fast=4.0), "fast_turns")])
def test_frequencies_refuse(args, match):
    rc, msg, _ = frequencies(**args)
    assert rc == TL_EINVAL and match in msg, (rc, msg)


@pytest.mark.parametrize("name,arguments", [
    ("rotary", 7), ("rotary_paged", 13), ("paged_attention", 10), ("pages_fork", 6), ("pages_extend", 6), ("pages_free", 6),
    ("pages_compact", 3), ("pages_copy", 5), ("beam_select", 8), ("beam_advance", 7)])
def test_native_front_end_takes_device_tensors_only(name, arguments):
    """The checks in front of the library, as far as they need no GPU: nothing but device tensors, all arguments there."""
    import torch
    from tensorlib_amd._lib import TensorLibError, front
    entry = getattr(front(), name)
    for wrong in (torch.zeros(2, 2), 1.5, None, "x"):
        with pytest.raises(TensorLibError, match="no CPU path"):
            entry(0, *[wrong] * (arguments - 1))
    with pytest.raises(TypeError, match=f"{arguments} arguments"):
        entry(0)
    with pytest.raises(TypeError, match=f"{arguments} arguments"):
        entry()
    with pytest.raises(TypeError, match="ordinal"):
        entry("0", *[None] * (arguments - 1))


# ------------------------------------------------------------------------------------------------ workspaces

def needed(name, args):
    """What a call asks for when its workspace is too small."""
    rc, msg = call(name, *args)
    assert rc == TL_EINVAL, (rc, msg)
    return int(re.search(r"workspace of (\d+) bytes", msg).group(1))


def attention_needs(n_seqs, n_heads, kv, dim, max_len):
    c = cache(page_stride=16 * kv * dim, row_stride=kv * dim, head_stride=dim, n_kv_heads=kv, head_dim=dim)
    args = changed(ATTENTION, cache=c, n_seqs=n_seqs, n_heads=n_heads, q_stride=n_heads * dim, max_len=max_len, ws=P, ws_bytes=0)
    exact = _lib.lib().tl_paged_attention_workspace_of_call(n_seqs, n_heads, kv, dim, max_len)
    if exact:           # then a call with none is refused; one that needs none would go on
        assert needed("tl_paged_attention_f16", args) == exact
    return exact


@pytest.mark.parametrize("n_heads,kv,dim", [(32, 8, 128), (32, 32, 128), (8, 1, 64), (40, 1, 96), (64, 8, 256), (4, 4, 8), (66, 2, 136)])
def test_an_attention_workspace_serves_every_smaller_call(n_heads, kv, dim):
    """Fewer sequences and shorter bounds take smaller chunks, so one call alone can need more than a larger one."""
    lib = _lib.lib()
    rng = np.random.RandomState(n_heads + dim)
    grew = False
    for max_seqs, limit in ((1, 131072), (1, 40000), (3, 9000), (17, 131072), (64, 4097), (200, 700), (1000, 33000), (5, 130), (9, 128)):
        enough = lib.tl_paged_attention_workspace(max_seqs, n_heads, kv, dim, limit)
        assert enough % (n_heads * (dim + 2) * 4) == 0
        lens = np.unique(np.concatenate([np.exp(rng.uniform(0, math.log(limit), 300)).astype(int), np.arange(1, limit // 128 + 1, max(1, limit // 128 // 300)) * 128, [limit]]))
        for n in {1, min(2, max_seqs), max_seqs // 2, max_seqs - 1, max_seqs} - {0}:
            largest = max(attention_needs(n, n_heads, kv, dim, int(x)) for x in lens if x <= limit)
            assert largest <= enough, (n, max_seqs, limit)
            grew |= largest > lib.tl_paged_attention_workspace_of_call(max_seqs, n_heads, kv, dim, limit)
    assert grew          # a call with a smaller bound did need more
    assert lib.tl_paged_attention_workspace(9, n_heads, kv, dim, 128) == 0


@pytest.mark.parametrize("args", [(0, 4, 2, 64, 100), (4, 0, 2, 64, 100), (4, 4, 0, 64, 100), (4, 4, 3, 64, 100), (4, 4, 2, 0, 100), (4, 4, 2, 64, 0), (-1, 4, 2, 64, 100)])
def test_workspaces_of_impossible_sizes(args):
    assert _lib.lib().tl_paged_attention_workspace(*args) == 0
    assert _lib.lib().tl_paged_attention_workspace_of_call(*args) == 0


@pytest.mark.parametrize("beams", [1, 4, 8, 64])
@pytest.mark.parametrize("vocab", [100, 8192, 8193, 32000, 100003, 300000])
def test_a_beam_workspace_serves_every_smaller_call(beams, vocab):
    """Few rows take shorter slices, so a call can need more than one with more rows."""
    lib = _lib.lib()
    for most in (1, 2, 5, 24, 100, 700):
        for n in (1, beams, min(64, beams * vocab)):
            enough = lib.tl_beam_select_workspace(most, beams, vocab, n)
            batches = sorted({1, 2, most} | set(range(1, most, max(1, most // 60)))) if most > 1 else [1]
            for smaller in (vocab, vocab // 2 + 1, max(n, vocab // 3)):
                for b in batches:
                    if b <= most and n <= beams * smaller:
                        assert needed("tl_beam_select_f16", changed(SELECT, n_batch=b, n_beams=beams, vocab=smaller, logits_stride=smaller, n_select=n, ws_bytes=0)) <= enough, (b, most, n)
