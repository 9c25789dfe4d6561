"""The cache's entry points without a GPU: what include/ntsamd_cache.h declares is exported, bad calls are refused before a
device is involved, empty ones succeed, and the dispatcher's choices (planning only)."""
import ctypes as C
import os
import re

import pytest
import torch

import niutensor_amd as nt

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 0x10000                                             # made up: no call below may follow it


def test_declared_and_exported():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "ntsamd_cache.h")).read(), flags=re.S)
    assert sorted(set(re.findall(r"\b(ntsamd_\w+)\s*\(", text))) == sorted(nt.CACHE_EXPORTS)
    lib = C.CDLL(nt.LIB_PATH)
    for name in nt.CACHE_EXPORTS:
        assert hasattr(lib, name), name


def make(dtype=3, pages=10, page=16, kv=2, dh=64, pool=None, pk=P, pv=P, n=3, width=4, tokens=3, new=1, length=0,
         lengths=P, starts=None, table=P):
    row = kv * dh
    cache = nt._Cache(pk, pv, dtype, pages, page, kv, dh, (C.c_longlong * 6)(*(pool or [page * row, row, dh] * 2)))
    return cache, nt._CacheBatch(lengths, starts, table, n, width, tokens, new, length)


def attend(q=P, out=P, heads=4, strides=(256, 64, 256, 64), prefix=None, null=None, **kw):
    cache, batch = make(**kw)
    st = (C.c_longlong * 4)(*strides) if strides else None
    a = (0, None, None if null == "cache" else C.byref(cache), None if null == "batch" else C.byref(batch), q, out, heads, st, 0.125, 1)
    L = nt.load()
    if prefix is not None:
        return L.ntsamd_attention_prefix(*a, prefix)
    return L.ntsamd_attention_cached(*a)


def append(k=P, v=P, q=P, q_out=P, heads=4, strides=(128, 64, 128, 64, 256, 64, 256, 64), rotation=P, positions=64, rotated=64,
           pairing=0, **kw):
    cache, batch = make(**kw)
    st = (C.c_longlong * 8)(*strides) if strides else None
    return nt.load().ntsamd_cache_append(0, None, C.byref(cache), C.byref(batch), k, v, q, q_out, heads, st, rotation, positions,
                                         rotated, pairing)


def message():
    return nt.load().ntsamd_last_error().decode()


@pytest.mark.parametrize("bad,code,text", [
    (dict(dtype=2, dh=6), 1, "head size"), (dict(dtype=4), 2, "Unsupported data type!"), (dict(dtype=0), 2, "Unsupported"),
    (dict(dh=136), 1, "head size"), (dict(dh=60), 1, "head size"), (dict(pages=-1), 1, "negative"), (dict(page=0), 1, "pages of 0"),
    (dict(n=-1), 1, "negative"), (dict(tokens=-1), 1, "negative"), (dict(new=-1), 1, "negative"), (dict(length=-1), 1, "negative"),
    (dict(pv=None), 1, "Empty"), (dict(lengths=None), 1, "Empty"), (dict(table=None), 1, "Empty"), (dict(pv=P + 8), 1, "16-byte"),
    (dict(lengths=P + 2), 1, "misaligned"), (dict(starts=P + 1), 1, "misaligned"),
    (dict(pool=[2048, 128, 60] * 2), 1, "multiples of 8"), (dict(pool=[-2048, 128, 64] * 2), 1, "non-negative"),
    (dict(pool=[2048, 64, 64] * 2), 1, "overlap"), (dict(pool=[1024, 128, 64] * 2), 1, "overlap"),
    (dict(length=65), 1, "4 pages of 16"), (dict(tokens=2), 1, "3 sequences of 1"), (dict(width=1 << 30, page=1 << 20, pool=[1 << 27, 128, 64] * 2), 1, "too large"),
])
def test_both_refuse(bad, code, text):
    assert attend(**bad) == code and text in message()
    assert append(**bad) == code and text in message()


@pytest.mark.parametrize("bad,text", [
    (dict(null="cache"), "Empty"), (dict(null="batch"), "Empty"), (dict(q=None), "Empty"), (dict(out=None), "Empty"), (dict(strides=None), "Empty"), (dict(heads=3), "evenly"),
    (dict(heads=-2), "negative"), (dict(q=P + 4), "16-byte"), (dict(out=P + 8), "16-byte"), (dict(strides=(250, 64, 256, 64)), "multiples"),
    (dict(strides=(256, 64, 192, 64)), "overlap"), (dict(strides=(256, 64, 256, 0)), "overlap"), (dict(prefix=-1), "prefix"),
])
def test_attention_refuses(bad, text):
    assert attend(**bad) == 1 and text in message()


@pytest.mark.parametrize("bad,text", [
    (dict(k=None), "Empty"), (dict(strides=None), "Empty"), (dict(q=None), "Empty"), (dict(q_out=None), "Empty"),
    (dict(rotated=63), "rotated"), (dict(rotated=66), "rotated"), (dict(rotated=-2), "rotated"), (dict(pairing=2), "pairing"),
    (dict(positions=-1), "negative"), (dict(heads=-1), "negative"), (dict(k=P + 1), "misaligned"), (dict(rotation=P + 2), "misaligned"),
    (dict(strides=(128, 64, 128, -64, 256, 64, 256, 64)), "negative"), (dict(strides=(128, 64, 128, 64, 256, 64, 128, 64)), "overlap"),
    (dict(strides=(128, 64, 128, 64, 256, 64, 64, 256)), "keep their strides"),
])
def test_append_refuses(bad, text):
    assert append(**bad) == 1 and text in message()


def test_nothing_to_do():
    for kw in (dict(n=0, tokens=0), dict(tokens=0, new=0), dict(new=0), dict(kv=0), dict(dh=0)):
        assert attend(**kw) == 0 and append(**kw) == 0
    assert attend(heads=0) == 0


def test_tensors_that_do_not_fit_are_refused():
    k = torch.zeros((4, 16, 2, 64), dtype=torch.float16)
    cache = nt.KVCache(k, k.clone())
    lens, table = torch.ones(3, dtype=torch.int32), torch.zeros((3, 4), dtype=torch.int32)
    batch = nt.CacheBatch(lens, table)
    q = torch.zeros((3, 4, 64), dtype=torch.float16)
    for bad in (torch.zeros((2, 4, 64), dtype=torch.float16), torch.zeros((3, 4, 32), dtype=torch.float16), q.float(), q[0],
                torch.zeros((3, 64, 4), dtype=torch.float16).transpose(1, 2)):
        with pytest.raises(nt.NtsAmdError):
            nt.attention_cached(cache, batch, q, bad, 1.0)
    with pytest.raises(nt.NtsAmdError, match="Unmatched"):
        nt.KVCache(k, k[:3])
    with pytest.raises(nt.NtsAmdError, match="columns"):
        nt.KVCache(k.transpose(2, 3).contiguous().transpose(2, 3), k.transpose(2, 3).contiguous().transpose(2, 3))
    with pytest.raises(nt.NtsAmdError, match="int32"):
        nt.CacheBatch(lens.long(), table)
    with pytest.raises(nt.NtsAmdError, match="Unmatched"):
        nt.CacheBatch(lens, table[:2])
    with pytest.raises(nt.NtsAmdError, match="Unmatched"):
        nt.CacheBatch(lens, table, starts=lens)
    with pytest.raises(nt.NtsAmdError, match="rotation"):
        nt.cache_append(cache, batch, q[:, :2], q[:, :2], rotation=torch.zeros((4, 32)))


@pytest.fixture()
def planning():
    nt.load()
    nt.tuning_set("NTSAMD_SPLIT_K", None)
    nt.plan_only(True)
    yield
    nt.plan_only(False)
    nt.tuning_set("NTSAMD_SPLIT_K", None)


def test_plans(planning):
    # short sequences: a workgroup takes a pair's keys alone, and nothing is joined
    assert attend(n=8, tokens=8, width=4) == 0 and nt.last_plan() == "attention_cached_kernel rows=16 whole=16"
    # long ones: in pieces
    assert attend(n=8, tokens=8, width=512) == 0
    assert re.fullmatch(r"attention_cached_kernel rows=16 pieces=\d+\+attention_join_kernel", nt.last_plan())
    # ones in between, or long ones without a workspace: whole, but by more waves
    assert attend(n=8, tokens=8, width=32) == 0 and nt.last_plan() == "attention_cached_kernel rows=16 wide whole=16"
    nt.tuning_set("NTSAMD_SPLIT_K", 1)
    assert attend(n=8, tokens=8, width=512) == 0 and nt.last_plan() == "attention_cached_kernel rows=16 wide whole=16"
    assert attend(n=8, tokens=8, width=512, prefix=1024) == 0 and nt.last_plan() == "attention_cached_kernel rows=16 wide whole=16"
    nt.tuning_set("NTSAMD_SPLIT_K", None)
    # the prefix once for all, each sequence's own keys, and the join
    assert attend(n=8, tokens=8, width=512, prefix=1024) == 0
    assert re.fullmatch(r"attention_prefix_kernel tiles=1x64 pieces=\d+ rows=16 pieces=\d+\+attention_join_kernel", nt.last_plan())
    # nothing to share
    assert attend(n=1, tokens=1, width=512, prefix=1024) == 0 and "prefix" not in nt.last_plan()
    assert attend(n=8, tokens=8, width=512, prefix=16) == 0 and "prefix" not in nt.last_plan()
    assert append() == 0 and nt.last_plan() == "cache_append_kernel"


def test_more_rows_than_a_launch_counts(planning):
    """500 million tokens of 4 query heads to a key head fit 31 bits, in tiles with one more for every sequence they do not."""
    big = dict(tokens=500000000, new=1000, width=64, starts=P, heads=8, strides=(512, 64, 512, 64))
    assert attend(n=1000, **big) == 0
    assert attend(n=1 << 22, **big) == 1 and "tensor too large" in message()
    assert attend(n=1000, **dict(big, tokens=600000000)) == 1 and "tensor too large" in message()
