"""The cache of keys and values on pages on the GPU (ntsamd_cache_append, ntsamd_attention_cached,
ntsamd_attention_prefix) against their definitions in 64 bits (tests/cache_reference.py, which derives the tolerances).
Everything in a pool that is no position of a sequence is NaN, so whatever is read beyond a sequence shows."""
import pytest

import niutensor_amd as nt
from cache_reference import Problem, assert_within, rotated_rows, rotation_table

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def name_the_case(request):
    print("\n[gpu-case] %s" % request.node.nodeid, flush=True)
    yield
    nt.tuning_set("NTSAMD_SPLIT_K", None)


# ---- appending -------------------------------------------------------------------------------------------------

APPEND = [
    # lens, new, heads, kv, dh, page, half, rotated, pairs, layout, uniform
    ([1], [1], 1, 1, 8, 1, True, 8, False, "rows", True),                          # the smallest there is
    ([128], [1], 8, 8, 64, 16, True, 64, False, "rows", True),
    ([33, 1, 257], [1, 1, 1], 32, 8, 128, 16, True, 128, False, "heads", True),
    ([33, 1, 257], [1, 1, 1], 6, 2, 96, 20, False, 32, True, "rows", True),
    ([40, 0, 70, 5, 300], [17, 0, 70, 1, 299], 8, 4, 64, 20, False, 64, False, "heads", False),
    ([40, 9, 70, 5, 300], [17, 0, 70, 0, 131], 4, 4, 80, 7, True, 40, True, "rows", False),
    ([9, 30], [9, 21], 2, 1, 24, 5, True, 12, False, "rows", False),               # 6 + 6 columns turned: pairs one by one
    ([9, 30], [9, 21], 2, 1, 20, 5, False, 6, True, "heads", False),
    ([200] * 130, [1] * 130, 2, 2, 32, 32, False, 0, False, "rows", False),        # more starts than a wave has lanes
    ([7, 8], [3, 3], 4, 2, 128, 4, True, None, False, "heads", True),              # no rotation at all
    ([30 + i % 5 for i in range(70)], [20 - i % 7 for i in range(70)], 8, 4, 64, 16, True, 64, False, "rows", False),   # many of both
    ([300, 310], [290, 300], 8, 4, 128, 16, False, 128, False, "heads", False),
]


@pytest.mark.parametrize("lens,new,heads,kv,dh,page,half,rotated,pairs,layout,uniform", APPEND)
def test_append(gpu, lens, new, heads, kv, dh, page, half, rotated, pairs, layout, uniform):
    import torch
    p = Problem(lens, new, heads, kv, dh, page, half, 3, layout, uniform=uniform, pad_tokens=0 if uniform else 3)
    cache, batch, q, out = p.place(nt)
    g = torch.Generator().manual_seed(8)
    both = torch.randn((p.tokens, 2 * kv, dh), generator=g).to(p.q.dtype)           # keys and values side by side
    k, v = both[:, :kv], both[:, kv:]
    bd = both.to(gpu)
    rot = rotation_table(max(lens), rotated) if rotated is not None else None
    want_k, want_v = p.k.double(), p.v.double()
    tol_k = torch.zeros_like(want_k)
    want_q, tol_q = torch.full(p.q.shape, 77.0, dtype=torch.float64), torch.zeros(p.q.shape, dtype=torch.float64)
    for i in range(len(lens)):
        a, b = p.starts[i], p.starts[i + 1]
        for t in range(a, b):
            pos = lens[i] - (b - a) + t - a
            page_, row = p.row(i, pos)
            cs = rot[pos:pos + 1] if rot is not None else torch.zeros((1, 0, 2))
            yk, ek = rotated_rows(k[t:t + 1], cs, pairs)
            yq, eq = rotated_rows(p.q[t:t + 1], cs, pairs)
            want_k[page_, row], tol_k[page_, row], want_v[page_, row] = yk[0], ek[0], v[t].double()
            want_q[t], tol_q[t] = yq[0], eq[0]
    nt.cache_append(cache, batch, bd[:, :kv], bd[:, kv:], rotation=rot.to(gpu) if rot is not None else None, pairs=pairs, q=q, q_out=out)
    for got, want, tol, what in ((p.kd, want_k, tol_k, "k"), (p.vd, want_v, torch.zeros_like(want_v), "v"), (out, want_q, tol_q, "q")):
        got = got.cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want)), what              # every other place as it was
        assert_within(torch.nan_to_num(got), torch.nan_to_num(want), tol, what)
    # the queries turned in place, keys and values not given twice: the same bits
    again = q.clone()
    nt.cache_append(cache, batch, bd[:, :kv], bd[:, kv:], rotation=rot.to(gpu) if rot is not None else None, pairs=pairs, q=again, q_out=again)
    own = p.starts[-1]
    assert torch.equal(again[:own], out[:own]) and torch.equal(again[own:], q[own:])


def test_append_rows_of_any_alignment(gpu):
    """Views that begin and step at odd elements take the way column by column: the same bits as dense ones."""
    import torch
    p = Problem([50, 20], [30, 2], 4, 2, 64, 16, True, 5)
    cache, batch, q, out = p.place(nt)
    rot = rotation_table(64, 64).to(gpu)
    k, v = torch.randn((32, 2, 64), device=gpu).half(), torch.randn((32, 2, 64), device=gpu).half()
    nt.cache_append(cache, batch, k, v, rotation=rot, q=q, q_out=out)
    k0, v0 = p.kd.clone(), p.vd.clone()

    def odd(x):
        big = torch.zeros((x.shape[0], x.shape[1], 71), dtype=x.dtype, device=gpu).flatten()
        y = big.as_strided(x.shape, (x.shape[1] * 71 - 1, 71, 1), 3)
        y.copy_(x)
        return y

    p.kd.fill_(float("nan"))
    p.vd.fill_(float("nan"))
    qo = odd(torch.zeros_like(q))
    nt.cache_append(cache, batch, odd(k), odd(v), rotation=rot, q=odd(q), q_out=qo)
    assert torch.equal(qo, out)
    wrote = ~torch.isnan(p.kd)
    assert int(wrote.sum()) == 32 * 2 * 64
    assert torch.equal(p.kd[wrote], k0[wrote]) and torch.equal(p.vd[wrote], v0[wrote])


def test_append_leaves_out_what_has_no_place(gpu):
    """Absent pages, positions before 0, past the table's row and past the rotation: nothing of them is written, and nothing else
    than the others' places."""
    import torch
    p = Problem([20, 20, 20, 20], [4, 4, 4, 4], 2, 2, 32, 8, False, 6, slack=0)
    p.table[0, 2] = 100000                                                         # absent: position 16 .. 19
    p.table[1, 2] = -1
    p.lens = [20, 20, 2, 26]                                                       # third: two tokens before 0; fourth: two past 3 pages
    p.max_length = 0
    cache, batch, q, out = p.place(nt)
    p.kd.fill_(float("nan"))
    p.vd.fill_(float("nan"))
    k, v = torch.ones((16, 2, 32), device=gpu), torch.ones((16, 2, 32), device=gpu)
    rot = rotation_table(24, 32).to(gpu)
    nt.cache_append(cache, batch, k, v, rotation=rot, q=q, q_out=out)
    wrote = (~torch.isnan(p.vd)).flatten(2).any(-1).cpu()                           # [pages, rows]
    want = torch.zeros_like(wrote)
    for i, pos in ((2, 0), (2, 1), (3, 22), (3, 23)):
        want[p.row(i, pos)] = True
    assert torch.equal(wrote, want)
    kept = (out == 77.0).flatten(1).all(-1).cpu().tolist()
    assert kept == [False] * 8 + [True, True, False, False] + [False, False, True, True]
    nt.cache_append(cache, batch, k, v, rotation=rot[:23], q=q, q_out=out.fill_(77.0))
    assert (out == 77.0).flatten(1).all(-1).cpu().tolist() == [False] * 8 + [True, True, False, False] + [False, True, True, True]


# ---- attention over the cache ------------------------------------------------------------------------------------

CACHED = [
    # lens, new, heads, kv, dh, page, half, causal, layout, uniform
    ([1], [1], 1, 1, 8, 1, True, True, "rows", True),
    ([1], [1], 1, 1, 4, 3, False, True, "rows", True),
    ([128], [1], 8, 8, 64, 16, True, True, "rows", True),
    ([31, 33, 64, 1, 0, 300], [1] * 6, 8, 2, 64, 16, True, True, "heads", True),
    ([31, 33, 64, 1, 0, 300], [1] * 6, 8, 2, 64, 16, False, True, "rows", True),
    ([700, 20, 1111], [1, 1, 1], 12, 4, 96, 20, True, True, "rows", True),
    ([700, 20, 1111], [1, 1, 1], 12, 4, 80, 7, False, True, "heads", True),
    ([5000], [1], 32, 8, 128, 64, True, True, "heads", True),                      # one sequence in pieces
    ([5000], [1], 4, 1, 128, 64, False, True, "heads", True),
    ([900, 2], [1, 1], 64, 2, 32, 16, True, True, "rows", True),                   # 32 query heads to a key head
    ([900, 2], [1, 1], 60, 1, 16, 100, True, True, "rows", True),                  # 60
    ([400, 2], [1, 1], 48, 2, 32, 16, False, True, "rows", True),                  # 24
    ([60, 70, 80], [3, 0, 5], 4, 2, 64, 16, True, True, "rows", False),            # a few tokens each, one with none
    ([60, 70, 800], [3, 0, 5], 4, 2, 128, 16, False, True, "heads", False),
    ([200, 64, 130, 77], [100, 64, 1, 40], 8, 4, 64, 16, True, True, "heads", False),    # pieces of text
    ([200, 64, 130, 77], [100, 64, 1, 40], 8, 4, 64, 20, False, True, "rows", False),
    ([300, 150], [33, 150], 6, 2, 128, 32, True, True, "rows", False),
    ([300, 150], [33, 150], 6, 2, 120, 32, True, True, "rows", False),
    ([1500], [40], 8, 2, 128, 16, True, True, "heads", False),                     # few tiles, long keys: tiles in pieces
    ([1500], [40], 8, 2, 36, 16, False, True, "heads", False),
    ([50, 3, 200, 0], [1, 40, 9, 2], 8, 8, 64, 16, False, False, "rows", False),   # not causal: more rows than keys, no keys
    ([50, 3, 200, 0], [1, 40, 9, 2], 8, 4, 64, 16, True, False, "heads", False),
    ([50, 3, 200, 17], [7] * 4, 8, 4, 40, 16, True, False, "rows", True),
]


@pytest.mark.parametrize("lens,new,heads,kv,dh,page,half,causal,layout,uniform", CACHED)
@pytest.mark.parametrize("bound", ["tight", "loose", "one piece"])
def test_cached(gpu, lens, new, heads, kv, dh, page, half, causal, layout, uniform, bound):
    p = Problem(lens, new, heads, kv, dh, page, half, 11, layout, uniform=uniform, pad_tokens=0 if uniform else 2,
                slack=3 if bound == "tight" else 400, max_length=0 if bound == "loose" else None)
    if bound == "one piece":
        nt.tuning_set("NTSAMD_SPLIT_K", 1)
    cache, batch, q, out = p.place(nt)
    want, tol = p.attention(causal)
    nt.attention_cached(cache, batch, q, out, p.scale, causal=causal)
    assert_within(out, want, tol, nt.last_plan())
    first = out.clone()
    nt.attention_cached(cache, batch, q, out.fill_(77.0), p.scale, causal=causal)
    assert (out == first).all()                                                    # the same bits on every run


TILES = [
    # sequences, positions, new tokens, heads, kv, dh, page, half, causal: the tiles' rows, and whether the keys are in pieces
    ((3, 70, 40, 64, 8, 80, 16, False, True), 32, False),
    ((4, 1000, 40, 8, 1, 128, 100, False, True), 32, True),
    ((8, 130, 120, 64, 8, 32, 20, False, True), 64, False),
    ((8, 130, 120, 64, 8, 64, 16, False, False), 64, False),
    ((8, 300, 250, 32, 4, 84, 16, False, True), 64, False),
    ((8, 300, 250, 64, 8, 128, 7, False, True), 64, False),
    ((4, 1700, 40, 64, 8, 96, 16, False, True), 64, True),
    ((3, 70, 40, 64, 8, 96, 16, True, False), 64, False),
    ((3, 1700, 900, 8, 2, 32, 16, True, True), 128, True),
    ((8, 70, 64, 64, 8, 64, 20, True, True), 128, False),
    ((8, 70, 64, 64, 8, 88, 16, True, False), 128, False),
    ((8, 70, 64, 64, 8, 128, 16, True, True), 128, False),
    ((8, 1700, 40, 4, 2, 96, 16, True, True), 16, True),
    ((1, 197, 42, 12, 4, 32, 20, True, True), 16, False),
    ((2, 568, 35, 16, 8, 64, 16, True, False), 16, False),
    ((3, 330, 33, 6, 3, 72, 7, True, True), 16, False),
    ((2, 300, 60, 8, 4, 128, 16, True, True), 16, False),
    ((3, 1100, 1000, 32, 8, 64, 16, True, True), 64, False),                      # more than run at once, long: the longest first
    ((3, 1100, 1000, 16, 8, 32, 16, False, False), 64, False),
]


@pytest.mark.parametrize("sizes,rows,pieces", TILES)
def test_every_kind_of_tile(gpu, sizes, rows, pieces):
    n, size, new, heads, kv, dh, page, half, causal = sizes
    p = Problem([size - 3 * i for i in range(n)], [new - 2 * i for i in range(n)], heads, kv, dh, page, half, 17,
                layout="heads" if dh % 32 else "rows", pad_tokens=1)
    cache, batch, q, out = p.place(nt)
    want, tol = p.attention(causal)
    nt.attention_cached(cache, batch, q, out, p.scale, causal=causal)
    assert "x%d pieces=" % rows in nt.last_plan() and pieces == ("join" in nt.last_plan()), nt.last_plan()
    assert_within(out, want, tol, nt.last_plan())


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("dh", [32, 64, 96, 128])
def test_long_keys_of_few_pairs_by_more_waves(gpu, half, dh):
    p = Problem([1021, 700, 0, 17, 512], [1] * 5, 6, 2, dh, 20, half, 18, uniform=True)
    cache, batch, q, out = p.place(nt)
    want, tol = p.attention(True)
    nt.tuning_set("NTSAMD_SPLIT_K", 1)
    nt.attention_cached(cache, batch, q, out, p.scale)
    assert "wide" in nt.last_plan(), nt.last_plan()
    assert_within(out, want, tol, nt.last_plan())


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("new", [1, 30])
@pytest.mark.parametrize("scale", [0.0, -0.2])
def test_scales_of_zero_and_below(gpu, half, new, scale):
    """Zero: the mean of what is seen; below: the smallest products weigh most."""
    p = Problem([90, 33, 30], [new] * 3, 4, 2, 64, 16, half, 19)
    p.scale = scale
    want, tol = p.attention(True)
    cache, batch, q, out = p.place(nt)
    nt.attention_cached(cache, batch, q, out, scale)
    assert_within(out, want, tol, nt.last_plan())


@pytest.mark.parametrize("half", [True, False])
def test_absent_pages_and_rows_that_see_nothing(gpu, half):
    """Positions on absent pages are left out; a sequence with none left, or more new tokens than positions, gives zeros there."""
    p = Problem([100, 48, 300, 3], [2, 1, 1, 5], 4, 2, 64, 16, half, 12)
    gone = [int(p.table[0, 1]), int(p.table[2, 0]), int(p.table[2, 18])] + [int(x) for x in p.table[1, :3]]
    want, tol = p.attention(True, absent=gone)
    assert (want[2] == 0).all() and (want[4:6] == 0).all()
    p.table[0, 1], p.table[2, 0], p.table[2, 18] = -1, 1 << 30, p.k.shape[0]
    p.table[1, :3] = -5
    cache, batch, q, out = p.place(nt)
    nt.attention_cached(cache, batch, q, out, p.scale)
    assert_within(out, want, tol, "absent pages")


@pytest.mark.parametrize("half", [True, False])
def test_large_scores(gpu, half):
    """Scores of several hundred: nothing overflows, one key or a few take it all."""
    p = Problem([500, 70], [1, 40], 4, 2, 128, 16, half, 13, spread=6.0)
    want, tol = p.attention(True)
    cache, batch, q, out = p.place(nt)
    nt.attention_cached(cache, batch, q, out, p.scale)
    assert_within(out, want, tol, "large scores")


def test_strided_queries_and_results(gpu):
    """q as part of a fused projection, out with gaps, which stay as they are."""
    import torch
    p = Problem([90, 40], [2, 1], 4, 2, 64, 16, True, 14)
    want, tol = p.attention(True)
    cache, batch, q, _ = p.place(nt)
    fused = torch.zeros((p.tokens, 8, 72), dtype=torch.float16, device=gpu)
    fused[:, :4, :64] = q
    big = torch.full((4, p.tokens, 88), 77.0, dtype=torch.float16, device=gpu)     # head by head
    out = big.transpose(0, 1)[:, :, 8:72]
    nt.attention_cached(cache, batch, fused[:, :4, :64], out, p.scale)
    assert_within(out, want, tol, "strided")
    assert (big[:, :, :8] == 77).all() and (big[:, :, 72:] == 77).all()


def test_pool_beyond_four_gigabytes(gpu):
    """Pages whose byte offsets pass 32 bits, in both directions of the cache."""
    import torch
    kv, dh, page, pages = 8, 128, 64, 40000                                         # 5.2 GB a pool
    kd = torch.zeros((pages, page, kv, dh), dtype=torch.float16, device=gpu)
    vd = torch.zeros((pages, page, kv, dh), dtype=torch.float16, device=gpu)
    cache = nt.KVCache(kd, vd)
    p = Problem([150, 100], [150, 100], 8, kv, dh, page, True, 15)
    want, tol = p.attention(True)
    where = {int(x): y for x, y in zip(p.table[p.table >= 0], (39999, 3, 20000, 35001, 39001))}
    table = torch.tensor([[where.get(int(x), -1) for x in row] for row in p.table], dtype=torch.int32)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)                 # noqa: E731
    batch = nt.CacheBatch(i32(p.lens), table.to(gpu), starts=i32(p.starts), tokens=p.tokens, max_new=p.max_new)
    k, v = torch.empty((250, kv, dh), dtype=torch.float16), torch.empty((250, kv, dh), dtype=torch.float16)
    for i in range(2):
        for t in range(p.lens[i]):
            k[p.starts[i] + t], v[p.starts[i] + t] = p.k[p.row(i, t)], p.v[p.row(i, t)]
    nt.cache_append(cache, batch, k.to(gpu), v.to(gpu))
    out = torch.full(p.q.shape, 77.0, dtype=torch.float16, device=gpu)
    nt.attention_cached(cache, batch, p.q.to(gpu), out, p.scale)
    assert_within(out, want, tol, "large pool")
    step = nt.CacheBatch(i32(p.lens), table.to(gpu))                                # the last token alone: the other kernel form
    last = torch.stack([p.q[149], p.q[249]])
    out = torch.full(last.shape, 77.0, dtype=torch.float16, device=gpu)
    nt.attention_cached(cache, step, last.to(gpu), out, p.scale)
    assert_within(out, want[[149, 249]], tol[[149, 249]], "large pool, one token")


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("new", [1, 20])
def test_pages_of_one_position_and_no_pages_at_all(gpu, half, new):
    import torch
    p = Problem([70, 20, 133], [new] * 3, 4, 2, 64, 1, half, 61, uniform=True)
    want, tol = p.attention(True)
    cache, batch, q, out = p.place(nt)
    nt.attention_cached(cache, batch, q, out, p.scale)
    assert_within(out, want, tol, nt.last_plan())
    none = nt.CacheBatch(p.lengths_d, p.table_d[:, :0].contiguous(), tokens=p.tokens, max_new=new)
    for prefix in (None, 64):
        out.fill_(77.0)
        if prefix is None:
            nt.attention_cached(cache, none, q, out, p.scale)
        else:
            nt.attention_prefix(cache, none, q, out, p.scale, prefix)
        assert (out == 0).all()                                                    # tokens that see nothing
    before = p.kd.clone()
    k = torch.ones((p.tokens, 2, 64), dtype=q.dtype, device=gpu)
    nt.cache_append(cache, none, k, k, q=q, q_out=out.fill_(77.0))
    assert torch.equal(torch.nan_to_num(p.kd), torch.nan_to_num(before)) and (out == 77).all()


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("new,prefix", [(1, None), (12, None), (1, 512)])
def test_more_rows_than_a_uniform_batch_has(gpu, half, new, prefix):
    p = Problem([600, 545, 570], [new] * 3, 8, 2, 64, 16, half, 62, prefix=prefix or 0, uniform=True, pad_tokens=5)
    want, tol = p.attention(True)
    cache, batch, q, out = p.place(nt)
    if prefix:
        nt.attention_prefix(cache, batch, q, out, p.scale, prefix)
    else:
        nt.attention_cached(cache, batch, q, out, p.scale)
    assert_within(out, want, tol, nt.last_plan())


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("new,prefix", [(1, None), (40, None), (1, 512)])
def test_lengths_and_starts_are_held_to_their_bounds(gpu, half, new, prefix):
    """A negative length is none, one beyond max_length is max_length, starts outside the rows end with them: every kernel holds what it
    reads to the bounds it was given, so that the other sequences come out right, and nothing else is touched."""
    import torch
    p = Problem([560, 550, 700, 640], [new] * 4, 8, 2, 64, 16, half, 63, prefix=prefix or 0, max_length=700, slack=0)
    want, tol = p.attention(True)
    cache, batch, q, out = p.place(nt)
    p.lengths_d.copy_(torch.tensor([560, -5, 2 ** 31 - 1, 640], dtype=torch.int32))
    p.starts_d[0], p.starts_d[4] = -7, 2 ** 30
    want[new:2 * new], tol[new:2 * new] = 0.0, 0.0
    if prefix:
        nt.attention_prefix(cache, batch, q, out, p.scale, prefix)
    else:
        nt.attention_cached(cache, batch, q, out, p.scale)
    assert_within(out, want, tol, nt.last_plan())


# ---- sequences with a common beginning ----------------------------------------------------------------------------

PREFIX = [
    # lens, new, heads, kv, dh, page, half, causal, prefix, layout, uniform
    ([130, 140, 150], [1, 1, 1], 8, 8, 64, 16, True, True, 128, "rows", True),
    ([130, 140, 150], [1, 1, 1], 8, 8, 64, 16, False, True, 128, "heads", True),
    ([513, 900, 512, 100, 0], [1] * 5, 8, 2, 128, 16, True, True, 512, "heads", True),     # shorter than the prefix, and empty
    ([513, 900, 512, 100, 0], [1] * 5, 8, 2, 128, 16, False, True, 512, "rows", True),
    ([700, 640, 777], [3, 0, 6], 12, 4, 96, 20, True, True, 640, "rows", False),
    ([700, 640, 777], [3, 0, 6], 12, 4, 36, 20, False, False, 640, "rows", False),
    ([2100, 2060], [40, 7], 4, 2, 64, 16, True, True, 2048, "rows", False),                # many rows: runs unshared
    ([300] * 70, [1] * 70, 4, 1, 64, 32, True, True, 288, "heads", False),                 # 280 rows against the prefix
    ([300] * 70, [1] * 70, 4, 1, 64, 32, False, True, 288, "heads", True),
    ([40, 41], [1, 1], 4, 4, 64, 16, True, True, 16, "rows", True),                        # too short to share
]


@pytest.mark.parametrize("lens,new,heads,kv,dh,page,half,causal,prefix,layout,uniform", PREFIX)
@pytest.mark.parametrize("bound", ["tight", "loose", "one piece"])
def test_prefix(gpu, lens, new, heads, kv, dh, page, half, causal, prefix, layout, uniform, bound):
    p = Problem(lens, new, heads, kv, dh, page, half, 21, layout, prefix=prefix, uniform=uniform, pad_tokens=0 if uniform else 2,
                slack=2 if bound == "tight" else 300, max_length=0 if bound == "loose" else None)
    if bound == "one piece":
        nt.tuning_set("NTSAMD_SPLIT_K", 1)
    cache, batch, q, out = p.place(nt)
    want, tol = p.attention(causal)
    nt.attention_prefix(cache, batch, q, out, p.scale, prefix, causal=causal)
    assert_within(out, want, tol, nt.last_plan())
    first = out.clone()
    nt.attention_prefix(cache, batch, q, out.fill_(77.0), p.scale, prefix, causal=causal)
    assert (out == first).all()


PREFIX_TILES = [
    # sequences, new tokens, prefix, heads, kv, dh, half: the tiles' rows
    ((60, 4, 1024, 4, 4, 32, False), 32),
    ((20, 4, 1024, 16, 2, 84, False), 32),
    ((20, 4, 512, 32, 8, 32, False), 64),
    ((20, 4, 1024, 32, 4, 64, False), 64),
    ((20, 4, 1024, 64, 8, 96, False), 64),
    ((20, 4, 1024, 64, 8, 128, False), 64),
    ((20, 4, 1024, 64, 8, 32, True), 128),
    ((60, 4, 1024, 32, 4, 64, True), 128),
    ((20, 4, 1024, 64, 8, 88, True), 128),
    ((60, 4, 1024, 32, 4, 128, True), 128),
]


@pytest.mark.parametrize("sizes,rows", PREFIX_TILES)
def test_every_kind_of_tile_of_the_prefix(gpu, sizes, rows):
    n, new, prefix, heads, kv, dh, half = sizes
    p = Problem([prefix + 40 - 2 * i if i != 3 else 300 for i in range(n)], [new - i % 3 for i in range(n)], heads, kv, dh, 32, half, 24,
                prefix=prefix, pad_tokens=2)
    cache, batch, q, out = p.place(nt)
    want, tol = p.attention(True)
    nt.attention_prefix(cache, batch, q, out, p.scale, prefix)
    assert "x%d pieces=" % rows in nt.last_plan() and "prefix" in nt.last_plan(), nt.last_plan()
    assert_within(out, want, tol, nt.last_plan())


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("n,prefix", [(62, 512), (64, 512), (64, 1024)])
def test_prefix_of_uneven_sequences(gpu, half, n, prefix):
    """62 do not fill the part and are cut into pieces; 64 are left whole. Behind 1024 positions they are more workgroups than run at
    once: the longest sequences come first, whichever place they have in the batch."""
    p = Problem([prefix + i * 37 % 300 for i in range(n)], [1] * n, 8, 8, 32, 16, half, 26, prefix=prefix, uniform=True)
    want, tol = p.attention(True)
    cache, batch, q, out = p.place(nt)
    nt.attention_prefix(cache, batch, q, out, p.scale, prefix)
    if prefix == 1024:
        assert "prefix" in nt.last_plan() and "whole=512" in nt.last_plan(), nt.last_plan()
    assert_within(out, want, tol, nt.last_plan())


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("prefix", [100, 1000, 1015])
def test_prefix_of_any_length(gpu, half, prefix):
    """A prefix need not end with a page: the page in which it ends is read through the first row for its part of it."""
    p = Problem([1030, 1100, 1015], [1, 1, 1], 4, 2, 64, 16, half, 25, prefix=1008, uniform=True)
    p.table[1:, 63] = p.table[0, 63]                                               # the rest of that page holds positions of all three
    want, tol = p.attention(True)
    cache, batch, q, out = p.place(nt)
    nt.attention_prefix(cache, batch, q, out, p.scale, prefix)
    assert_within(out, want, tol, nt.last_plan())


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("prefix", [1010, 1012, 1015])
@pytest.mark.parametrize("new,heads,kv", [(1, 4, 2), (40, 4, 2), (120, 32, 4)])
@pytest.mark.parametrize("dh", [32, 64, 128])
def test_page_in_which_a_prefix_ends(gpu, half, prefix, new, heads, kv, dh):
    """Every sequence has a page of its own there, of which only what follows the prefix counts; one or many new tokens."""
    p = Problem([1060, 1100, 1071], [new] * 3, heads, kv, dh, 16, half, 27, prefix=1008)
    p.row = lambda i, pos: (int(p.table[0 if pos < prefix else i, pos // 16]), pos % 16)
    want, tol = p.attention(True)
    cache, batch, q, out = p.place(nt)
    nt.attention_prefix(cache, batch, q, out, p.scale, prefix)
    assert_within(out, want, tol, nt.last_plan())


def test_prefix_is_read_through_the_first_row_of_the_table(gpu):
    """The other sequences' entries for the prefix are not looked at."""
    p = Problem([140, 150, 160], [1, 1, 1], 4, 2, 64, 16, True, 22, prefix=128, uniform=True)
    want, tol = p.attention(True)
    p.table[1:, :8] = -1
    cache, batch, q, out = p.place(nt)
    nt.attention_prefix(cache, batch, q, out, p.scale, 128)
    assert_within(out, want, tol, "first row")


@pytest.mark.parametrize("uniform", [True, False])
def test_prefix_of_more_sequences_than_one_workspace_takes(gpu, uniform):
    """Thousands of sequences go through the workspace in slices."""
    n = 2300
    p = Problem([130 + i % 40 for i in range(n)], [1] * n, 8, 8, 128, 32, True, 23, prefix=128, uniform=uniform)
    want, tol = p.attention(True)
    cache, batch, q, out = p.place(nt)
    nt.attention_prefix(cache, batch, q, out, p.scale, 128)
    assert_within(out, want, tol, nt.last_plan())


# ---- together, as a program uses them ------------------------------------------------------------------------------

@pytest.mark.parametrize("half", [True, False])
def test_a_generation_from_prompt_to_tokens(gpu, half):
    """Prompts enter the cache in one call and attend to themselves, then step by step one token each: at every step
    the result is the attention, in 64 bits, over the rotated keys of all positions so far."""
    import torch
    n, heads, kv, dh, page, steps = 3, 4, 2, 64, 16, 5
    prompt = [37, 5, 64]
    dt = torch.float16 if half else torch.float32
    total = [a + steps for a in prompt]
    p = Problem(total, [a for a in prompt], heads, kv, dh, page, half, 31)
    rot = rotation_table(max(total), dh)
    g = torch.Generator().manual_seed(1)
    rows = [[torch.randn((total[i], h, dh), generator=g).to(dt) for h in (heads, kv, kv)] for i in range(n)]
    kd, vd = torch.full(p.k.shape, float("nan"), dtype=dt, device=gpu), torch.full(p.v.shape, float("nan"), dtype=dt, device=gpu)
    cache = nt.KVCache(kd, vd)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)                 # noqa: E731
    lengths, rd = i32(prompt), rot.to(gpu)
    table = p.table.to(gpu)
    done = [0] * n
    for step in range(steps + 1):
        new = prompt if step == 0 else [1] * n
        cat = lambda j: torch.cat([rows[i][j][done[i]:done[i] + new[i]] for i in range(n)])          # noqa: E731
        q, k, v = cat(0).to(gpu), cat(1).to(gpu), cat(2).to(gpu)
        if step == 0:
            starts = i32([0, 37, 42, 106])
            batch = nt.CacheBatch(lengths, table, starts=starts, tokens=106, max_new=64)
        elif step == 1:
            batch = nt.CacheBatch(lengths, table)
        if step > 0:
            lengths += 1
        nt.cache_append(cache, batch, k, v, rotation=rd, q=q, q_out=q)
        out = torch.empty_like(q)
        nt.attention_cached(cache, batch, q, out, dh ** -0.5)
        for i in range(n):
            done[i] += new[i]
        # the same through the definition: rotated rows rounded to the type, as they stand in the cache
        r = Problem(done, new, heads, kv, dh, page, half, 31)
        r.table = p.table
        r.k, r.v = torch.full(p.k.shape, float("nan"), dtype=dt), torch.full(p.k.shape, float("nan"), dtype=dt)
        r.q = q.cpu()
        for i in range(n):
            exact, err = rotated_rows(rows[i][1][:done[i]], rot[:done[i]], False)
            for t in range(done[i]):
                got = kd[p.row(i, t)].cpu()
                assert_within(got, exact[t], err[t], "key %d of %d" % (t, i))
                r.k[p.row(i, t)], r.v[p.row(i, t)] = got, rows[i][2][t]
        want, tol = r.attention(True)
        assert_within(out, want, tol, "step %d" % step)


def test_recorded_and_replayed_with_other_lengths(gpu):
    """One step - append, attention, attention with a shared prefix - recorded once and replayed while the sequences
    grow, with eager work between the replays; every replay gives the eager call's bits."""
    import torch
    n, heads, kv, dh, page = 5, 8, 2, 128, 16
    p = Problem([600, 520, 900, 513, 700], [1] * n, heads, kv, dh, page, True, 41, prefix=512, uniform=True, slack=8, max_length=0)
    cache, batch, q, out = p.place(nt)
    for i in range(n):                                                             # room for the steps to come
        used = -(-p.lens[i] // page)
        p.table_d[i, used:used + 2] = torch.tensor([0, 0], dtype=torch.int32)
    spare = torch.zeros((2 * n, page, kv, dh), dtype=torch.float16, device=gpu)
    p.kd, p.vd = torch.cat([p.kd, spare]), torch.cat([p.vd, spare])
    p.kd.nan_to_num_()                                                             # the lengths run ahead of what is appended
    p.vd.nan_to_num_()
    first = p.k.shape[0]
    for i in range(n):
        used = -(-p.lens[i] // page)
        p.table_d[i, used], p.table_d[i, used + 1] = first + 2 * i, first + 2 * i + 1
    cache = nt.KVCache(p.kd, p.vd)
    rot = rotation_table(1200, dh).to(gpu)
    k, v = torch.randn((n, kv, dh), device=gpu).half(), torch.randn((n, kv, dh), device=gpu).half()
    q0 = q.clone()
    shared = torch.empty_like(out)

    def step():
        nt.cache_append(cache, batch, k, v, rotation=rot, q=q0, q_out=q)
        nt.attention_cached(cache, batch, q, out, p.scale)
        nt.attention_prefix(cache, batch, q, shared, p.scale, 512)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
    for turn in range(6):
        k.normal_()
        v.normal_()
        q0.normal_()
        out.zero_()
        shared.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone(), shared.clone(), q.clone()
        step()
        torch.cuda.synchronize()
        assert torch.equal(got[0], out) and torch.equal(got[1], shared) and torch.equal(got[2], q), turn
        assert ((out.float() - shared.float()).abs() <= 2.0 ** -8 * 4).all()        # two roundings of probabilities and results of size below 4
        p.lengths_d += 5


def test_streams_and_released_workspaces(gpu):
    """Calls on two streams at once have their own workspaces; a release between calls costs an allocation, no more."""
    import torch
    p = Problem([3000, 100], [1, 1], 8, 2, 128, 16, True, 51)
    want, tol = p.attention(True)
    cache, batch, q, out = p.place(nt)
    outs = [torch.full_like(out, 77.0) for _ in range(8)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i, o in enumerate(outs):
        with torch.cuda.stream(streams[i % 2]):
            nt.attention_cached(cache, batch, q, o, p.scale)
    torch.cuda.synchronize()
    for o in outs:
        assert_within(o, want, tol, "two streams")
    nt.release_workspaces()
    nt.attention_cached(cache, batch, q, out, p.scale)
    assert_within(out, want, tol, "after a release")


def test_two_host_threads_on_one_stream(gpu):
    """Both threads' calls share the stream's workspace: neither's pieces get between the other's kernels."""
    import threading
    import torch
    problems = [Problem([3000, 100, 2500], [1, 1, 1], 8, 2, 128, 16, True, 71), Problem([2000, 700], [30, 40], 8, 2, 64, 16, False, 72),
                Problem([1300, 1400, 1290], [1, 1, 1], 8, 2, 64, 16, True, 73, prefix=1280, uniform=True)]
    jobs = []
    for p in problems:
        cache, batch, q, _ = p.place(nt)
        jobs.append((p, cache, batch, q, [torch.full_like(q, 77.0) for _ in range(15)], p.attention(True)))
    torch.cuda.synchronize()
    failed = []

    def work(p, cache, batch, q, outs, _, prefix):
        try:
            for o in outs:
                if prefix:
                    nt.attention_prefix(cache, batch, q, o, p.scale, prefix)
                else:
                    nt.attention_cached(cache, batch, q, o, p.scale)
        except Exception as e:                          # noqa: BLE001 - the main thread reports it
            failed.append(e)

    threads = [threading.Thread(target=work, args=(*j, prefix)) for j, prefix in zip(jobs, (0, 0, 1280))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed
    for p, _, _, _, outs, (want, tol) in jobs:
        for o in outs:
            assert_within(o, want, tol, "threads")


@pytest.mark.parametrize("half", [True, False])
def test_pieces_of_text_recorded_and_replayed(gpu, half):
    """Prompts appended and attended to in tiles, recorded with room for longer ones and replayed with other lengths and starts."""
    import torch
    heads, kv, dh, page = 8, 2, 64, 16
    sizes = [([700, 300, 900], [200, 100, 212]), ([900, 280, 640], [30, 270, 212]), ([512, 513, 900], [170, 171, 171])]
    p = Problem([900] * 3, [200, 100, 212], heads, kv, dh, page, half, 74)
    cache, batch, q, out = p.place(nt)
    p.kd.nan_to_num_()
    p.vd.nan_to_num_()
    batch = nt.CacheBatch(p.lengths_d, p.table_d, starts=p.starts_d, tokens=512, max_new=300, max_length=900)
    k, v = torch.randn((512, kv, dh), device=gpu).to(q.dtype), torch.randn((512, kv, dh), device=gpu).to(q.dtype)

    def step():
        nt.cache_append(cache, batch, k, v)
        nt.attention_cached(cache, batch, q, out, p.scale)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
    for turn in range(2):
        for lens, new in sizes:
            starts = [0]
            for a in new:
                starts.append(starts[-1] + a)
            p.lengths_d.copy_(torch.tensor(lens, dtype=torch.int32))
            p.starts_d.copy_(torch.tensor(starts, dtype=torch.int32))
            k.normal_()
            out.fill_(77.0)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            got = out.clone()
            p.lens, p.new, p.starts, p.tokens = lens, new, starts, 512
            p.k, p.v = p.kd.cpu(), p.vd.cpu()
            want, tol = p.attention(True)
            assert_within(got, want, tol, "replay %d" % turn)
            step()
            torch.cuda.synchronize()
            assert torch.equal(got, out)
