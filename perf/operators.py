"""The cache operators as they are measured: their cases, their inputs, their plain forms and their results in 64 bits.

Three operators of serving with a cache of keys and values that stands in pages:
  append   keys and values of new tokens go to their sequences' pages, keys (and queries) rotated by their position on the way
  cached   attention of the new tokens to everything their sequence has in the cache
  prefix   the same for sequences that begin with the same keys and values, which are read once for all of them

A case: dtype; seqs sequences whose lengths run from len_min to len_max and that have new_min to new_max new tokens each;
heads query heads over kv key heads of dh columns; pages of `page` positions, stored position by position ("rows") or head
by head ("heads"); rot rotated columns, as halves or as neighbours ("pairs"); prefix positions in common.
"""
import math

import torch

own = False

DTYPES = {"half": torch.float16, "float": torch.float32}
BASE = 10000.0


def _case(name, op, dtype, seqs, len_min, len_max, new_min, new_max, heads, kv, dh, page, layout, rot=0, pairs=False,
          causal=True, prefix=0):
    c = dict(name=name, op=op, dtype=dtype, seqs=seqs, len_min=len_min, len_max=len_max, new_min=new_min, new_max=new_max,
             heads=heads, kv=kv, dh=dh, page=page, layout=layout)
    if op == "append":
        c.update(rot=rot, pairs=pairs)
    else:
        c.update(causal=causal)
    if op == "prefix":
        c.update(prefix=prefix)
    return c


def listed():
    return [
        # one sentence being decoded, base model of 8 heads of 64: a call is all latency
        _case("append_step_1_half", "append", "half", 1, 77, 77, 1, 1, 8, 8, 64, 16, "rows", rot=64),
        # a server's step: 64 sequences, one token each, four query heads to a key head
        _case("append_steps_64_half", "append", "half", 64, 33, 257, 1, 1, 32, 8, 128, 16, "heads", rot=128),
        # a few inputs of odd lengths in float, neighbouring columns rotated, part of the head only
        _case("append_ragged_7_float", "append", "float", 7, 300, 701, 1, 499, 8, 8, 64, 20, "rows", rot=32, pairs=True),
        # prompts entering the cache
        _case("append_prompts_8_half", "append", "half", 8, 1024, 2048, 513, 2048, 32, 8, 128, 64, "heads", rot=128),
        # one sentence being decoded
        _case("cached_step_1_half", "cached", "half", 1, 128, 128, 1, 1, 8, 8, 64, 16, "rows"),
        # a batch of sentences being decoded in float, lengths as they come
        _case("cached_steps_32_float", "cached", "float", 32, 9, 1021, 1, 1, 8, 8, 64, 16, "rows"),
        # a server's step: 64 sequences from just begun to long
        _case("cached_steps_64_half", "cached", "half", 64, 1, 8191, 1, 1, 32, 8, 128, 16, "heads"),
        # one very long document, one token at a time: few rows, a long axis
        _case("cached_step_long_half", "cached", "half", 1, 131072, 131072, 1, 1, 32, 8, 128, 64, "heads"),
        # pieces of prompts against what is in the cache before them
        _case("cached_chunks_4_half", "cached", "half", 4, 1500, 4096, 257, 1024, 32, 8, 128, 64, "heads"),
        # target rows against the cached states of their source sentences: every row sees the whole source
        _case("cached_cross_16_float", "cached", "float", 16, 5, 200, 1, 40, 8, 8, 64, 16, "rows", causal=False),
        # the hypotheses of one sentence behind a common prompt
        _case("prefix_beams_8_float", "prefix", "float", 8, 513, 601, 1, 1, 8, 8, 64, 16, "rows", prefix=512),
        # many requests with the same long instructions before their own text
        _case("prefix_64_half", "prefix", "half", 64, 8193, 8704, 1, 1, 32, 8, 128, 16, "heads", prefix=8192),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        most[c["op"]] = (max(most.get(c["op"], (0, 0))[0], w["bytes"]), max(most.get(c["op"], (0, 0))[1], w["flops"]))
    op = rng.choice(["append", "cached", "cached", "prefix"])
    dtype = rng.choice(["half", "half", "float"])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 8])
    dh = rng.choice([32, 64, 64, 80, 96, 128, 128])
    page = rng.choice([8, 16, 16, 32, 64, 20, 100, 128])
    layout = rng.choice(["rows", "heads"])
    seqs = _log(rng, 1, 128)
    few = rng.random() < 0.6                            # steps of one token, or pieces of text
    rot = rng.choice([dh, dh, dh // 2 // 8 * 8])
    pairs = rng.random() < 0.4
    causal = rng.random() < 0.75
    prefix = 0
    if op == "append":
        top = 1 if few else _log(rng, 2, 2048)
        len_max = top + _log(rng, 1, 256)
    else:
        top = 1 if few else _log(rng, 2, 1024)
        len_max = _log(rng, max(top, 16), 16384)
    if op == "prefix":
        top = 1 if few else rng.randint(2, 6)
        prefix = max(1, _log(rng, 64, 16384) // page) * page
        len_max = prefix + top + _log(rng, 1, 512)
    case = None
    while True:
        new_min = max(1, top // 4)
        least = prefix + top if op == "prefix" else top
        len_max = max(len_max, least)
        case = _case("", op, dtype, seqs, max(least, min(len_max, least + (len_max - least) // 7)), len_max, new_min, top,
                     heads, kv, dh, page, layout, rot, pairs, causal, prefix)
        w = work(case)
        # the keys of every sequence, gathered: no more than the largest listed case has
        gathered = seqs * len_max * kv * dh
        if w["bytes"] <= most[op][0] and w["flops"] <= max(most[op][1], 1) and gathered <= 64 * 8704 * 8 * 128:
            break
        if seqs > 1:
            seqs = max(1, seqs * 2 // 3)
        elif heads > kv:
            heads = kv
        else:
            top = max(1, top // 2)
            len_max = max(1, len_max // 2)
            prefix = max(1, prefix // 2 // page) * page if op == "prefix" else 0
    del case["name"]
    return case


def _spread(lo, hi, n):
    """n whole numbers from lo to hi, evenly spread."""
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _sizes(case):
    """Length and number of new tokens of every sequence, in no particular order of their own."""
    n = case["seqs"]
    lens = _spread(case["len_min"], case["len_max"], n)
    new = _spread(case["new_min"], case["new_max"], n)
    new = [new[(i * 5 + 3) % n] for i in range(n)] if n % 5 else new
    least = case.get("prefix", 0)
    return lens, [max(1, min(a, b - least)) for a, b in zip(new, lens)]


def prepare(case, seed):
    dev = torch.device("cuda")
    dt = DTYPES[case["dtype"]]
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    gc = torch.Generator()
    gc.manual_seed(seed)
    lens, new = _sizes(case)
    order = torch.randperm(len(lens), generator=gc).tolist()
    lens, new = [lens[i] for i in order], [new[i] for i in order]
    n, page, kv, dh, heads = case["seqs"], case["page"], case["kv"], case["dh"], case["heads"]
    tokens, shared = sum(new), case.get("prefix", 0) // page
    need = [-(-a // page) for a in lens]
    pages = shared + sum(a - shared for a in need) + 3
    perm = torch.randperm(pages, generator=gc).to(torch.int32)
    table = torch.zeros((n, max(need)), dtype=torch.int32)
    at = shared
    for i, a in enumerate(need):
        table[i, :shared] = perm[:shared]
        table[i, shared:a] = perm[at:at + a - shared]
        at += a - shared
    normal = lambda *shape: torch.randn(shape, generator=g, device=dev, dtype=dt)  # noqa: E731
    # the cache as [page][position in the page][head][column], however it is stored
    pool = lambda: (normal(pages, page, kv, dh) if case["layout"] == "rows"  # noqa: E731
                    else normal(pages, kv, page, dh).transpose(1, 2))
    s = dict(case=dict(case), k_cache=pool(), v_cache=pool(), table=table.to(dev), tokens=tokens, max_new=max(new), max_length=max(lens),
             lengths=torch.tensor(lens, dtype=torch.int32, device=dev))
    starts = [0]
    for a in new:
        starts.append(starts[-1] + a)
    # one token for every sequence needs no starts
    s["starts"] = None if case["new_max"] == 1 else torch.tensor(starts, dtype=torch.int32, device=dev)
    s["q"] = normal(tokens, heads, dh)
    s["out"] = torch.empty((tokens, heads, dh), dtype=dt, device=dev)
    s["scale"] = dh ** -0.5
    if case["op"] == "append":
        # keys and values as the projection leaves them: side by side in one tensor
        kv_new = normal(tokens, 2 * kv, dh)
        s["k"], s["v"] = kv_new[:, :kv], kv_new[:, kv:]
        ang = _angles(torch.arange(max(lens), device=dev), case["rot"])
        s["rotation"] = torch.stack((ang.cos(), ang.sin()), -1).float().contiguous()
    if own:
        import niutensor_amd as nt
        s["cache"] = nt.KVCache(s["k_cache"], s["v_cache"])
        s["batch"] = nt.CacheBatch(s["lengths"], s["table"], starts=s["starts"], tokens=tokens, max_new=s["max_new"],
                                   max_length=s["max_length"])
    return s


def _angles(pos, rot):
    """position / BASE^(2 j / rot), in 64 bits."""
    j = torch.arange(rot // 2, device=pos.device, dtype=torch.float64)
    return pos.double()[:, None] * torch.exp(j * (-2.0 * math.log(BASE) / rot))


def _own(s):
    import niutensor_amd as nt
    c = s["case"]
    if c["op"] == "append":
        nt.cache_append(s["cache"], s["batch"], s["k"], s["v"], rotation=s["rotation"], pairs=c["pairs"], q=s["q"], q_out=s["out"])
        return {"k_cache": s["k_cache"], "v_cache": s["v_cache"], "q": s["out"]}
    if c["op"] == "cached":
        nt.attention_cached(s["cache"], s["batch"], s["q"], s["out"], s["scale"], causal=c["causal"])
    else:
        nt.attention_prefix(s["cache"], s["batch"], s["q"], s["out"], s["scale"], c["prefix"], causal=c["causal"])
    return {"out": s["out"]}


def run(s):
    if own:
        return _own(s)
    return _plain_append(s) if s["case"]["op"] == "append" else _plain_attention(s)


def _tokens(s):
    """Sequence, place among its sequence's new tokens, and position of every token; new tokens of every sequence."""
    n, dev = s["case"]["seqs"], s["lengths"].device
    starts = s["starts"].long() if s["starts"] is not None else torch.arange(n + 1, device=dev)
    new = starts[1:] - starts[:-1]
    t = torch.arange(s["tokens"], device=dev)
    seq = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    place = t - starts[seq]
    return starts, new, seq, place, s["lengths"].long()[seq] - new[seq] + place


def _rotate(x, cs, pairs):
    """The first columns of x [tokens, heads, dh] turned by (cos, sin) [tokens, columns / 2, 2], in 32 bits, rounded once."""
    h = cs.shape[1]
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    y = x.float()
    a, b = (y[..., 0:2 * h:2], y[..., 1:2 * h:2]) if pairs else (y[..., :h], y[..., h:2 * h])
    u, w = a * c - b * s, b * c + a * s
    turned = torch.stack((u, w), -1).flatten(-2) if pairs else torch.cat((u, w), -1)
    return torch.cat((turned, y[..., 2 * h:]), -1).to(x.dtype)


def _plain_append(s):
    c = s["case"]
    _, _, seq, _, pos = _tokens(s)
    page, row = s["table"][seq, pos // c["page"]].long(), pos % c["page"]
    cs = s["rotation"][pos]
    s["k_cache"][page, row] = _rotate(s["k"], cs, c["pairs"])
    s["v_cache"][page, row] = s["v"]
    s["out"].copy_(_rotate(s["q"], cs, c["pairs"]))
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"], "q": s["out"]}


def _plain_attention(s):
    c = s["case"]
    n, kv, dh, heads, most = c["seqs"], c["kv"], c["dh"], c["heads"], s["max_new"]
    per, dev = heads // kv, s["q"].device
    starts, new, seq, place, _ = _tokens(s)
    pos = torch.arange(s["max_length"], device=dev)
    page = s["table"].long()[:, pos // c["page"]]
    k = s["k_cache"][page, (pos % c["page"])[None]].float().permute(0, 2, 3, 1)                # sequence, head, column, position
    v = s["v_cache"][page, (pos % c["page"])[None]].float().permute(0, 2, 1, 3)
    at = (starts[:-1, None] + torch.arange(most, device=dev)).clamp(max=s["tokens"] - 1)
    q = s["q"].float()[at].reshape(n, most, kv, per, dh).permute(0, 2, 1, 3, 4).reshape(n, kv, most * per, dh)
    lens = s["lengths"].long()
    seen = lens[:, None].expand(n, most)
    if c["causal"]:
        seen = (lens - new + 1)[:, None] + torch.arange(most, device=dev)
    hidden = pos >= seen.repeat_interleave(per, 1)[:, None, :, None]
    hidden = hidden | (pos >= lens[:, None, None, None])
    x = torch.matmul(q, k.contiguous()).mul_(s["scale"]).masked_fill_(hidden, -math.inf)
    x = x.sub_(x.amax(-1, keepdim=True)).exp_()
    y = torch.matmul(x, v.contiguous()) / x.sum(-1, keepdim=True)
    y = y.reshape(n, kv, most, per, dh).permute(0, 2, 1, 3, 4).reshape(n, most, heads, dh)
    s["out"].copy_(y[seq, place])
    return {"out": s["out"]}


def work(case):
    lens, new = _sizes(case)
    size = DTYPES[case["dtype"]].itemsize
    heads, kv, dh, tokens = case["heads"], case["kv"], case["dh"], sum(new)
    if case["op"] == "append":
        # every new row of k, v and q read and written; the rows of the rotation
        return {"bytes": 2 * tokens * (2 * kv + heads) * dh * size + tokens * case["rot"] * 4,
                "flops": tokens * (kv + heads) * case["rot"] * 3}
    shared = case.get("prefix", 0)
    keys = shared + sum(a - shared for a in lens)
    seen = sum(a * b - (b * (b - 1) // 2 if case["causal"] else 0) for a, b in zip(lens, new))
    return {"bytes": keys * kv * dh * 2 * size + 2 * tokens * heads * dh * size, "flops": 4 * dh * heads * seen}


def exact(case, seed):
    s = prepare(case, seed)
    lens, table = s["lengths"].tolist(), s["table"].tolist()
    n, page, kv, dh = case["seqs"], case["page"], case["kv"], case["dh"]
    starts = s["starts"].tolist() if s["starts"] is not None else list(range(n + 1))
    if case["op"] == "append":
        kc, vc, q = s["k_cache"].double(), s["v_cache"].double(), s["q"].double()
        k, v, h = s["k"].double(), s["v"].double(), case["rot"] // 2
        first, second = ((slice(0, 2 * h, 2), slice(1, 2 * h, 2)) if case["pairs"] else (slice(0, h), slice(h, 2 * h)))
        for i in range(n):
            a, b = starts[i], starts[i + 1]
            pos = torch.arange(lens[i] - (b - a), lens[i], device=q.device)
            z = torch.polar(torch.ones((), dtype=torch.float64, device=q.device), _angles(pos, case["rot"]))[:, None]
            for x in (k, q):                            # a pair of columns is a complex number, the rotation a product
                y = torch.complex(x[a:b, :, first], x[a:b, :, second]) * z
                x[a:b, :, first], x[a:b, :, second] = y.real, y.imag
            where = torch.tensor([table[i][p // page] for p in pos.tolist()], device=q.device)
            kc[where, pos % page], vc[where, pos % page] = k[a:b], v[a:b]
        return {"k_cache": kc, "v_cache": vc, "q": q}
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for i in range(n):
        a, b, size = starts[i], starts[i + 1], lens[i]
        ids = torch.tensor(table[i][:-(-size // page)], device=out.device)
        for h in range(kv):
            k = s["k_cache"][ids, :, h].reshape(-1, dh)[:size].double()
            v = s["v_cache"][ids, :, h].reshape(-1, dh)[:size].double()
            r = slice(h * (case["heads"] // kv), (h + 1) * (case["heads"] // kv))
            x = torch.tensordot(s["q"][a:b, r].double(), k, ([2], [1])) * dh ** -0.5             # token, head, position
            if case["causal"]:
                last = torch.arange(size - (b - a), size, device=out.device)
                x.masked_fill_(torch.arange(size, device=out.device) > last[:, None, None], -math.inf)
            out[a:b, r] = torch.tensordot(torch.softmax(x, -1), v, ([2], [0]))
    return {"out": out}
