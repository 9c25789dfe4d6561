"""The cache's operators at the limits of what a batch may hold: what stands beyond a sequence's end, whatever its bits, in a prefix that
others share. Against the definitions in 64 bits (tests/cache_reference.py)."""
import math

import pytest

import niutensor_amd as nt
from cache_reference import Problem, assert_within

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def name_the_case(request):
    print("\n[gpu-case] %s" % request.node.nodeid, flush=True)
    yield
    nt.tuning_set("NTSAMD_SPLIT_K", None)


# ---- a prefix of which some sequences have a part only ------------------------------------------------------------

BEHIND = [
    # sequences, new tokens, prefix, heads, kv, dh, half: rows of the prefix's tiles
    ((6, 1, 512, 4, 4, 32, False), 16),
    ((6, 1, 512, 4, 4, 128, False), 16),
    ((6, 4, 2048, 32, 4, 64, False), 32),
    ((6, 4, 2048, 64, 8, 96, False), 32),
    ((20, 4, 1024, 32, 4, 64, False), 64),
    ((20, 4, 512, 64, 8, 128, False), 64),
    ((6, 1, 512, 4, 4, 64, True), 64),
    ((6, 1, 520, 4, 4, 128, True), 64),
    ((20, 4, 2048, 32, 4, 96, True), 128),
    ((20, 4, 2048, 64, 8, 64, True), 128),
]


@pytest.mark.parametrize("sizes,rows", BEHIND)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("short", ["some", "the first", "all"])
@pytest.mark.parametrize("bound", ["tight", "loose"])
def test_what_a_prefix_holds_beyond_a_sequence(gpu, sizes, rows, bad, short, bound):
    """From position `end` on the prefix is not finite. Sequences that end there or before never see it, whoever shares the prefix, and
    with nobody there who has it all."""
    n, new, prefix, heads, kv, dh, half = sizes
    end = prefix // 3 + 7
    lens = [(end, 0, end - 1, 1, end // 64 * 64, end // 2)[i % 6] if short == "all" or (i % 2 == 0) == (short == "the first") else prefix + 30 - i
            for i in range(n)]
    p = Problem(lens, [new] * n, heads, kv, dh, 8, half, 81, layout="heads" if dh % 64 else "rows", prefix=prefix, uniform=new == 1, pad_tokens=1,
                slack=prefix // 8 + (8 if bound == "tight" else 400), max_length=prefix + 30 if bound == "tight" else 0)
    for at in range(end, prefix):
        page, row = p.row(0, at)
        p.k[page, row], p.v[page, row] = bad, bad
    cache, batch, q, out = p.place(nt)
    nt.attention_prefix(cache, batch, q, out, p.scale, prefix)
    assert "prefix" in nt.last_plan() and (bound == "loose" or "x%d pieces=" % rows in nt.last_plan()), nt.last_plan()
    want, tol = p.attention(True)
    mine = [t for i in range(n) if lens[i] <= end for t in range(p.starts[i], p.starts[i + 1])] + [p.tokens - 1]
    assert_within(out[mine], want[mine], tol[mine], nt.last_plan())


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("new", [1, 3])
def test_sequences_that_have_any_part_of_a_prefix(gpu, half, new):
    """Lengths around every border of the prefix's pieces and blocks, all finite, with and without a causal limit; own keys in pieces."""
    prefix = 1000
    lens = [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 192, 250, 256, 257, 320, 384, 500, 512, 513, 640, 768, 769, 896, 960, 961, 998, 999, 1000,
            1001, 1063, 2500]
    p = Problem(lens, [new] * len(lens), 8, 4, 64, 8, half, 82, prefix=prefix)
    for causal in (True, False):
        want, tol = p.attention(causal)
        cache, batch, q, out = p.place(nt)
        nt.attention_prefix(cache, batch, q, out, p.scale, prefix, causal=causal)
        assert "prefix" in nt.last_plan() and "pieces" in nt.last_plan().split()[-1], nt.last_plan()
        assert_within(out, want, tol, nt.last_plan())


FINITE = [
    # the tiles of a prefix that a few rows make: sequences, new tokens, prefix, heads, kv, dh, half: rows of a tile
    ((6, 1, 1000, 4, 4, 32, False), 16),
    ((3, 1, 2048, 8, 2, 128, False), 16),
    ((2, 2, 700, 6, 2, 88, False), 16),
    ((6, 1, 1000, 4, 4, 32, True), 64),
    ((3, 1, 2048, 8, 2, 128, True), 64),
    ((2, 2, 700, 6, 2, 88, True), 64),
]


@pytest.mark.parametrize("sizes,rows", FINITE)
def test_tiles_of_a_prefix_for_few_rows(gpu, sizes, rows):
    n, new, prefix, heads, kv, dh, half = sizes
    p = Problem([prefix + 50 - 7 * i for i in range(n)], [new] * n, heads, kv, dh, 20, half, 90, prefix=prefix, pad_tokens=1)
    p.row = lambda i, pos: (int(p.table[0 if pos < prefix else i, pos // 20]), pos % 20)       # 2048 ends inside a page
    want, tol = p.attention(True)
    cache, batch, q, out = p.place(nt)
    nt.attention_prefix(cache, batch, q, out, p.scale, prefix)
    assert "prefix" in nt.last_plan() and "x%d pieces=" % rows in nt.last_plan(), nt.last_plan()
    assert_within(out, want, tol, nt.last_plan())


@pytest.mark.parametrize("half", [True, False])
def test_sequences_that_grow_past_a_prefix_in_a_replay(gpu, half):
    """Recorded while all sequences end inside the prefix, replayed until all have it."""
    import torch
    p = Problem([300, 511, 20, 512, 480], [1] * 5, 8, 2, 64, 16, half, 91, prefix=512, uniform=True, slack=8, max_length=640)
    own = torch.arange(40, dtype=torch.int32).view(5, 8)
    p.table[:, 32:40] = p.k.shape[0] + own
    more = [torch.randn((40, 16, 2, 64), generator=torch.Generator().manual_seed(i)).to(p.k.dtype) for i in (1, 2)]
    p.k, p.v = torch.cat([p.k, more[0]]), torch.cat([p.v, more[1]])
    for i in range(1, 5):                               # the reference goes by every sequence's own row
        p.table[i, :32] = p.table[0, :32]
    cache, batch, q, out = p.place(nt)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        nt.attention_prefix(cache, batch, q, out, p.scale, 512)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            nt.attention_prefix(cache, batch, q, out, p.scale, 512)
    for lens in ([300, 511, 20, 512, 480], [400, 512, 0, 513, 511], [512, 600, 513, 639, 512], [1, 63, 64, 65, 640]):
        p.lens = lens
        p.lengths_d.copy_(torch.tensor(lens, dtype=torch.int32))
        out.fill_(77.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want, tol = p.attention(True)
        assert_within(out, want, tol, str(lens))


# ---- batches of different sequences ------------------------------------------------------------------------------------

@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,new", [
    ([2000, 1500, 17, 900, 1], [1, 1, 1, 200, 1]),      # steps of one token beside a piece of text
    ([300, 2200, 64], [300, 2, 64]),                    # prompts, whose positions are all new, beside a step of two
    ([513, 257, 128, 1], [513, 257, 128, 1]),           # prompts alone
])
def test_batches_of_different_sequences(gpu, half, causal, lens, new):
    p = Problem(lens, new, 8, 2, 64, 16, half, 94, pad_tokens=1)
    want, tol = p.attention(causal)
    cache, batch, q, out = p.place(nt)
    nt.attention_cached(cache, batch, q, out, p.scale, causal=causal)
    assert_within(out, want, tol, nt.last_plan())


# ---- pools and rows in other orders ------------------------------------------------------------------------------------

@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("order", ["keys and values side by side", "positions first", "heads first", "padded rows"])
@pytest.mark.parametrize("new,page", [(1, 16), (40, 16), (40, 20), (40, 8), (40, 2)])
def test_pools_in_any_order(gpu, half, order, new, page):
    import torch
    p = Problem([130, 64, 97], [new] * 3, 8, 2, 64, page, half, 92)
    cache, batch, q, out = p.place(nt)
    if order == "keys and values side by side":
        both = torch.stack([p.k, p.v], 1).to(gpu)       # [pages][2][positions][heads][columns]
        p.kd, p.vd = both[:, 0], both[:, 1]
    elif order == "padded rows":
        p.kd, p.vd = (torch.nn.functional.pad(x, (0, 8, 0, 1), value=float("nan")).to(gpu)[:, :, :2, :64] for x in (p.k, p.v))
    else:
        turn = (1, 0, 2, 3) if order == "positions first" else (2, 0, 1, 3)
        back = [turn.index(i) for i in range(4)]
        p.kd, p.vd = (x.permute(turn).contiguous().to(gpu).permute(back) for x in (p.k, p.v))
    cache = nt.KVCache(p.kd, p.vd)
    want, tol = p.attention(True)
    nt.attention_cached(cache, batch, q, out, p.scale)
    assert_within(out, want, tol, nt.last_plan())
    k = torch.randn((p.tokens, 2, 64), device=gpu).to(q.dtype)
    nt.cache_append(cache, batch, k, k)
    for i in range(3):
        for t in (0, new - 1):
            page_, row = p.row(i, p.lens[i] - new + t)
            assert torch.equal(p.kd[page_, row], k[p.starts[i] + t]) and torch.equal(p.vd[page_, row], k[p.starts[i] + t])


@pytest.mark.parametrize("new", [1, 40])
def test_queries_and_rows_that_stand_for_many(gpu, new):
    """Strides of zero: one query for all heads, one row of values for all tokens."""
    import torch
    p = Problem([130, 64], [new] * 2, 8, 2, 64, 16, True, 93)
    p.q = p.q[:, :1].expand(-1, 8, -1).contiguous()
    want, tol = p.attention(True)
    cache, batch, q, out = p.place(nt)
    nt.attention_cached(cache, batch, q[:, :1].contiguous().expand(-1, 8, -1), out, p.scale)
    assert_within(out, want, tol, nt.last_plan())
    k, v = torch.randn((1, 1, 64), device=gpu).half().expand(p.tokens, 2, 64), torch.randn((1, 2, 64), device=gpu).half().expand(p.tokens, 2, 64)
    nt.cache_append(cache, batch, k, v)
    for i in range(2):
        page, row = p.row(i, p.lens[i] - 1)
        assert torch.equal(p.kd[page, row], k[0]) and torch.equal(p.vd[page, row], v[0])


# ---- probabilities in half -----------------------------------------------------------------------------------------

@pytest.mark.parametrize("new,heads,slack,split,plan", [
    (1, 8, 2, None, "rows=16 whole="), (1, 8, 400, None, "rows=16 pieces="), (1, 8, 400, 1, "rows=16 wide whole="),
    (4, 16, 2, None, "rows=32 whole="), (4, 16, 400, None, "rows=32 pieces="), (35, 4, 2, None, "attention_cached_tile_kernel tiles=")])
@pytest.mark.parametrize("dh", [32, 64, 128])
def test_few_rows_in_half_lose_no_bits_of_the_probabilities(gpu, new, heads, slack, split, plan, dh):
    """They go into the second product as the sum of two halves: the first leaves 2^-11 of a probability at most, the second 2^-11 of
    that, or 2^-25 where it is below the normal range, of probabilities whose sum, in fp32, is at least 1. So beside what fp32 leaves,
    (2^-22 + 2^-25 n) max |v| and the rounding of the result, which is 2^-11 of it or 2^-25."""
    p = Problem([64, 40, 47], [new] * 3, heads, 2, dh, 16, True, 89, slack=slack, max_length=0)
    nt.tuning_set("NTSAMD_SPLIT_K", split)
    cache, batch, q, out = p.place(nt)
    nt.attention_cached(cache, batch, q, out, p.scale)
    assert plan in nt.last_plan(), nt.last_plan()
    p.half = False                                      # the tolerance of fp32
    want, tol = p.attention(True)
    most = float(p.v.nan_to_num().abs().max())
    tol = (tol + (2.0 ** -22 + 2.0 ** -25 * 64) * most) * (1 + 2.0 ** -10) + (2.0 ** -11 * want.abs()).clamp(min=2.0 ** -25) * (1 + 2.0 ** -10)
    assert_within(out, want, tol, nt.last_plan())


# ---- batches without new tokens ------------------------------------------------------------------------------------

@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("max_new,prefix,plan", [(1, 0, "pieces="), (1, 512, "attention_prefix_kernel"), (40, 0, "tiles=")])
@pytest.mark.parametrize("start", [0, 2])
def test_a_batch_without_new_tokens(gpu, half, max_new, prefix, plan, start):
    """All starts equal: nothing is computed, and no row is touched. One sequence with a token among such ones gets its result."""
    n = 5
    p = Problem([3000, 2900, 2000, 1024, 600], [1] * n, 8, 2, 64, 16, half, 83, prefix=prefix, pad_tokens=40)
    p.max_new = max_new
    cache, batch, q, out = p.place(nt)
    call = (lambda: nt.attention_prefix(cache, batch, q, out, p.scale, prefix)) if prefix else (lambda: nt.attention_cached(cache, batch, q, out, p.scale))
    p.starts_d.fill_(start)
    call()
    assert plan in nt.last_plan(), nt.last_plan()
    assert (out == 77.0).all()
    before = p.kd.clone()
    new = q[:, :2].contiguous()
    nt.cache_append(cache, batch, new, new)
    assert (p.kd == before).logical_or(before.isnan()).all() and (p.kd.isnan() == before.isnan()).all()
    p.starts_d[3:] = start + 1
    call()
    p.new, p.starts = [0, 0, 1, 0, 0], [start] * 3 + [start + 1] * 3
    want, tol = p.attention(True)
    assert_within(out, want, tol, nt.last_plan())


# ---- tables of nothing ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("positions,rotated", [(0, 64), (0, 0), (50, 0)])
def test_a_rotation_of_nothing(gpu, positions, rotated):
    """Tokens beyond its positions are left out, as with any other; the others are stored as they are where no columns are turned."""
    import torch
    p = Problem([60, 30, 51], [20, 2, 1], 4, 2, 64, 16, True, 87)
    cache, batch, q, out = p.place(nt)
    p.kd.fill_(5.0)
    p.vd.fill_(5.0)
    k, v = torch.ones((23, 2, 64), dtype=torch.float16, device=gpu), torch.ones((23, 2, 64), dtype=torch.float16, device=gpu)
    nt.cache_append(cache, batch, k, v, rotation=torch.zeros((positions, rotated // 2, 2), device=gpu), q=q, q_out=out)
    at = [*range(40, 60), 28, 29, 50]
    seq = [0] * 20 + [1] * 2 + [2]
    want = torch.full(p.k.shape, 5.0, dtype=torch.float16)
    for t in range(23):
        if at[t] < positions:
            want[p.row(seq[t], at[t])] = 1.0
    assert torch.equal(p.kd.cpu(), want) and torch.equal(p.vd.cpu(), want)
    there = torch.tensor([x < positions for x in at], device=gpu)
    assert torch.equal(out[there], q[there]) and (out[~there] == 77.0).all()


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("new,prefix", [(1, 0), (40, 0), (1, 512)])
def test_a_scale_that_is_not_a_number(gpu, half, new, prefix):
    """Every score is one, and so is every result (a scale of zero would give the mean)."""
    p = Problem([600, 545, 570], [new] * 3, 8, 2, 64, 16, half, 88, prefix=prefix)
    cache, batch, q, out = p.place(nt)
    if prefix:
        nt.attention_prefix(cache, batch, q, out, math.nan, prefix)
    else:
        nt.attention_cached(cache, batch, q, out, math.nan)
    assert out.isnan().all()


# ---- more workgroups than a launch may have ---------------------------------------------------------------------------

def test_more_tokens_than_a_launch_takes(gpu):
    """2^26 and some tokens of one row of keys and of values: a wave each, four to a workgroup, of which a launch has 2^24 at most."""
    import torch
    tokens, page = (1 << 26) + 77, 1 << 16
    pages = -(-tokens // page)
    kd, vd = (torch.zeros((pages, page, 1, 4), device=gpu) for _ in range(2))
    k, v = (torch.arange(tokens * 4, dtype=torch.int32, device=gpu).view(torch.float32).view(tokens, 1, 4) for _ in range(2))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)                 # noqa: E731
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(84))
    batch = nt.CacheBatch(i32([tokens]), order.to(torch.int32).to(gpu)[None], tokens=tokens, max_new=tokens)
    nt.cache_append(nt.KVCache(kd, vd), batch, k, v)
    for got, put in ((kd, k), (vd, v)):
        got = got[order.to(gpu)].view(-1, 1, 4)
        assert torch.equal(got[:tokens].view(torch.int32), put.view(torch.int32)) and (got[tokens:] == 0).all()


@pytest.mark.parametrize("length", [1, 300])
def test_more_sequences_than_a_launch_takes(gpu, length):
    """2^24 and some sequences of one token, all on the same pages; short ones are left whole, long ones cut into pieces and joined."""
    import torch
    n, page = (1 << 24) + 3, 300
    g = torch.Generator().manual_seed(85)
    k, v = (torch.randn((1, page, 1, 8), generator=g).half() for _ in range(2))
    kinds = torch.randn((64, 1, 8), generator=g).half()
    cache = nt.KVCache(k.to(gpu), v.to(gpu))
    batch = nt.CacheBatch(torch.full((n,), length, dtype=torch.int32, device=gpu), torch.zeros((n, 1), dtype=torch.int32, device=gpu))
    q = kinds.to(gpu).repeat(n // 64 + 1, 1, 1)[:n].contiguous()
    out = torch.full_like(q, 77.0)
    nt.attention_cached(cache, batch, q, out, 0.5)
    p = Problem([length], [1], 1, 1, 8, page, True, 85, uniform=True)
    p.k, p.v, p.scale, p.table = k, v, 0.5, p.table * 0
    for i in range(64):
        p.q = kinds[i:i + 1]
        want, tol = p.attention(True)
        lo, hi = (want - tol).to(gpu), (want + tol).to(gpu)
        assert ((out[i::64].double() >= lo) & (out[i::64].double() <= hi)).all(), i


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("uniform", [True, False])
def test_more_sequences_than_a_launch_cuts_into_pieces(gpu, half, uniform):
    n = 4500
    p = Problem([1400 if i % 450 == 449 else 3 + i % 40 for i in range(n)], [1] * n if uniform else [i % 3 for i in range(n)], 2, 1, 8, 16, half, 86,
                uniform=uniform)
    want, tol = p.attention(True)
    cache, batch, q, out = p.place(nt)
    nt.attention_cached(cache, batch, q, out, p.scale)
    assert " pieces=" in nt.last_plan(), nt.last_plan()
    assert_within(out, want, tol, nt.last_plan())
