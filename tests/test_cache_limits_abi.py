"""What a call of the cache's entry points may hold at most, without a GPU (planning only): calls that no launch takes are refused before
the first one."""
import ctypes as C

import pytest

import niutensor_amd as nt

P = 0x10000                                             # made up: no call below may follow it


@pytest.fixture(autouse=True)
def planning():
    nt.load()
    nt.tuning_set("NTSAMD_SPLIT_K", None)
    nt.plan_only(True)
    yield
    nt.plan_only(False)
    nt.tuning_set("NTSAMD_SPLIT_K", None)


def call(what, heads, n=1, tokens=1, new=1, kv=1, dh=8, page=16, width=4, dtype=3, starts=None, odd=0):
    row = kv * dh
    cache = nt._Cache(P, P, dtype, 10, page, kv, dh, (C.c_longlong * 6)(*[page * row, row, dh] * 2))
    batch = nt._CacheBatch(P, starts, P, n, width, tokens, new, 0)
    L = nt.load()
    if what == "append":
        st = (C.c_longlong * 8)(row, dh, row, dh, heads * dh, dh, heads * dh, dh)
        rc = L.ntsamd_cache_append(0, None, C.byref(cache), C.byref(batch), P + odd, P, P, P, heads, st, None, 0, 0, 0)
    else:
        st = (C.c_longlong * 4)(heads * dh, dh, heads * dh, dh)
        rc = L.ntsamd_attention_cached(0, None, C.byref(cache), C.byref(batch), P, P, heads, st, 0.125, 1)
    return rc, L.ntsamd_last_error().decode() if rc else nt.last_plan()


def test_workgroups_of_tiles():
    """256 threads to a workgroup, fewer than 2^32 threads to a launch: 2^23 tiles of two key heads are one too many."""
    rc, plan = call("attention", 8, tokens=(1 << 28) - 32, new=(1 << 28) - 32, kv=2)
    assert rc == 0 and "tiles=%dx128 pieces=1" % ((1 << 23) - 1) in plan
    rc, text = call("attention", 8, tokens=1 << 28, new=1 << 28, kv=2)
    assert rc == 1 and "tensor too large" in text


def test_pairs_go_in_slices():
    for n in ((1 << 24) + 3, 1 << 28):
        assert call("attention", 1, n=n, tokens=n)[0] == 0
        assert call("attention", 1, n=n, tokens=n, width=400)[0] == 0
    rc, text = call("attention", 1 << 24, kv=1 << 24, tokens=1)
    assert rc == 1 and "tensor too large" in text


def test_sequences_in_pieces_go_in_slices():
    """Every workgroup looks at all sequences of its launch, so that a launch of many takes the square of their time."""
    rc, plan = call("attention", 1, n=1 << 16, tokens=1 << 16, width=400)
    assert rc == 0 and int(plan.split("pieces=")[1].split("+")[0]) <= 2048 + 512


def test_items_of_a_token():
    """The kernel counts a token's items in 31 bits; tokens go in slices."""
    assert call("append", 1 << 29)[0] == 0
    for heads, odd in (((1 << 31) - 1, 0), (1 << 29, 2)):
        rc, text = call("append", heads, odd=odd)
        assert rc == 1 and "tensor too large" in text
    rc, text = call("append", 1, kv=(1 << 31) - 1)
    assert rc == 1 and "tensor too large" in text
    assert call("append", 1, tokens=(1 << 31) - 1, new=(1 << 31) - 1)[0] == 0


def test_numbers_beyond_32_bits_are_refused_by_the_binding():
    import torch
    lengths, table = torch.ones(2, dtype=torch.int32), torch.zeros((2, 4), dtype=torch.int32)
    for kw in (dict(tokens=(1 << 32) + 2), dict(max_new=(1 << 32) + 1, tokens=2), dict(max_length=1 << 32), dict(max_length=(1 << 32) + 7)):
        with pytest.raises(nt.NtsAmdError, match="32 bits"):
            nt.CacheBatch(lengths, table, **kw)
    k = torch.zeros((4, 16, 2, 64), dtype=torch.float16)
    q = torch.zeros((2, 4, 64), dtype=torch.float16)
    with pytest.raises(nt.NtsAmdError, match="32 bits"):
        nt.attention_prefix(nt.KVCache(k, k.clone()), nt.CacheBatch(lengths, table), q, q.clone(), 1.0, (1 << 32) + 16)
    wide = torch.zeros(1, dtype=torch.float16).expand((1 << 32) + 3, 16, 2, 1)
    with pytest.raises(nt.NtsAmdError, match="32 bits"):
        nt.KVCache(wide, wide)


def test_a_result_without_queries_is_refused_by_the_binding():
    import torch
    k = torch.zeros((4, 16, 2, 64), dtype=torch.float16)
    batch = nt.CacheBatch(torch.ones(2, dtype=torch.int32), torch.zeros((2, 4), dtype=torch.int32))
    new, q = torch.zeros((2, 2, 64), dtype=torch.float16), torch.zeros((2, 4, 64), dtype=torch.float16)
    with pytest.raises(nt.NtsAmdError, match="queries"):
        nt.cache_append(nt.KVCache(k, k.clone()), batch, new, new, q_out=q)
