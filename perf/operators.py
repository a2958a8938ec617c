"""What is measured of the operators that decode several candidates of a chunk: attention over a prefix that a group of
rows shares, the pages that hold every candidate's own tokens, and the penalties and masks on their logits.

``run`` computes an operator in its plain form (elementary torch operations) or, with ``own`` set, through this package's entry
points (``viktor_b200.ops``).  Sizes are those of this repository's decoder (8 query / 2 KV heads of 64, prefixes up to 2049
positions, tails up to 1100 tokens, the 343-token vocabulary) and generic ones of larger models."""

import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
INF = float("inf")


# ------------------------------------------------------------------------------------------------------ cases
def _attend(name, dtype, heads, kv_heads, dim, groups, each, ragged, prefix_lo, prefix, tail_lo, tail, page, pad):
    """groups x each rows (ragged: sizes spread around ``each``, some groups empty); prefix lengths spread over
    prefix_lo..prefix, tails over tail_lo..tail; ``pad`` rows behind the last group."""
    return dict(name=name, op="attend", dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, groups=groups, each=each,
                ragged=ragged, prefix_lo=prefix_lo, prefix=prefix, tail_lo=tail_lo, tail=tail, page=page, pad=pad)


def _fork(name, layers, page, kv_heads, dim, parents, children, lo, hi):
    """``children`` rows become copies of ``parents`` rows whose lengths spread over lo..hi."""
    return dict(name=name, op="fork", layers=layers, page=page, kv_heads=kv_heads, dim=dim, parents=parents,
                children=children, lo=lo, hi=hi)


def _compact(name, layers, page, kv_heads, dim, pages, rows, live):
    """A pool of ``pages`` pages of which ``live`` per cent are used, scattered."""
    return dict(name=name, op="compact", layers=layers, page=page, kv_heads=kv_heads, dim=dim, pages=pages, rows=rows,
                live=live)


def _start(name, page, rows, count, pages):
    """All rows given up and room made for ``count`` tokens in each."""
    return dict(name=name, op="start", page=page, rows=rows, count=count, pages=pages)


def _penal(name, dtype, rows, vocab, tokens, mask, bias):
    """Penalties by up to ``tokens`` tokens of each row; ``mask`` grammar states (0: no mask); a bias or none."""
    return dict(name=name, op="penal", dtype=dtype, rows=rows, vocab=vocab, tokens=tokens, mask=mask, bias=bias)


def listed():
    return [
        # four candidates of two short chunks just after the start: the latency of a call
        _attend("attend small", "bf16", 8, 2, 64, 2, 4, False, 100, 200, 1, 16, 16, 0),
        # an engine batch of 256 chunks, four candidates each, in the middle of their decoding
        _attend("attend chunks", "bf16", 8, 2, 64, 256, 4, False, 400, 2049, 1, 1100, 64, 0),
        # one long prompt for a whole batch of a larger model: bound by the products
        _attend("attend one prompt", "f16", 32, 8, 128, 1, 256, False, 32768, 32768, 1, 512, 64, 0),
        # few rows on a very long prefix without shared heads: the long axis has to be split
        _attend("attend few rows", "f16", 16, 16, 64, 1, 4, False, 131071, 131071, 1, 33, 16, 0),
        # uneven groups, some of them empty, rows and prefixes without tokens, odd head ratio, padded batch
        _attend("attend ragged", "bf16", 12, 2, 128, 37, 9, True, 0, 1501, 0, 300, 32, 7),
        # a beam step of two chunks
        _fork("fork small", 8, 16, 2, 64, 2, 6, 3, 40),
        # 256 chunks get seven more candidates each
        _fork("fork batch", 8, 64, 2, 64, 256, 1792, 1, 900),
        # a pool after many candidates have ended at odd times
        _compact("compact pool", 8, 64, 2, 64, 6000, 1024, 45),
        # a new batch of candidates takes the place of the last one
        _start("start batch", 16, 2048, 40, 9001),
        # the 4-mer vocabulary at the end of a chunk, every state with its grammar mask
        _penal("penal 4-mers", "f32", 256, 343, 1100, 5, True),
        # a batch of a large vocabulary
        _penal("penal large", "f32", 512, 131072, 2048, 64, True),
        # odd sizes, bf16 logits, no grammar
        _penal("penal odd", "bf16", 33, 50021, 4097, 0, False),
    ]


def _spread(rng, lo, hi):
    """A whole number of lo..hi, evenly over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "fork", "compact", "start", "penal", "penal"])
    if op == "attend":
        heads, kv_heads, dim = rng.choice([(8, 2, 64), (8, 2, 64), (32, 8, 128), (16, 16, 64), (12, 2, 128), (8, 1, 64),
                                           (6, 3, 128), (16, 1, 128)])
        ragged = rng.random() < 0.4
        groups, each = _spread(rng, 1, 256), _spread(rng, 1, 256)
        prefix, tail = _spread(rng, 1, 131072), _spread(rng, 1, 1100)
        prefix_lo, tail_lo = (0, 0) if ragged else (max(1, prefix // rng.randint(1, 8)), 1)
        c = _attend(None, rng.choice(["bf16", "f16"]), heads, kv_heads, dim, groups, each, ragged, prefix_lo, prefix,
                    tail_lo, tail, rng.choice([16, 32, 64, 128]), rng.randint(0, 9) if ragged else 0)
        while work(c)["bytes"] > 3.5e8 or work(c)["flops"] > 1.2e11 or c["groups"] * c["each"] > 2048:
            # the axis that is furthest from its start goes first
            k = max(("groups", "each", "prefix", "tail"), key=lambda k: c[k] / {"groups": 4, "each": 8, "prefix": 256,
                                                                                "tail": 64}[k])
            c[k] = max(1, c[k] * 2 // 3)
            c["prefix_lo"] = min(c["prefix_lo"], c["prefix"])
        del c["name"]
        return c
    if op == "fork":
        parents = _spread(rng, 1, 256)
        hi = _spread(rng, 1, 1100)
        c = _fork(None, rng.choice([1, 3, 8]), rng.choice([16, 32, 64, 128]), rng.choice([1, 2, 8]), rng.choice([64, 128]),
                  parents, _spread(rng, 1, 7 * parents), rng.randint(0, hi), hi)
        while work(c)["bytes"] > 4e8:
            c["children"] = c["children"] // 2
    elif op == "compact":
        c = _compact(None, rng.choice([1, 3, 8]), rng.choice([16, 32, 64]), rng.choice([1, 2, 8]), rng.choice([64, 128]),
                     _spread(rng, 8, 6000), 0, rng.randint(5, 95))
        while c["layers"] * c["page"] * c["kv_heads"] * c["dim"] * c["pages"] > 3.9e8:
            c["pages"] = c["pages"] // 2
        c["rows"] = _spread(rng, 1, max(1, c["pages"] // 6))
    elif op == "start":
        page, rows, count = rng.choice([16, 32, 64]), _spread(rng, 1, 2048), _spread(rng, 1, 64)
        c = _start(None, page, rows, count, rows * -(-count // page) + rng.randint(1, 3000))
    else:
        c = _penal(None, rng.choice(["f32", "f32", "bf16", "f16"]), _spread(rng, 1, 512), _spread(rng, 7, 131072),
                   _spread(rng, 1, 4097), rng.choice([0, 1, 7, 64]), rng.random() < 0.5)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------------------ inputs
def _even(lo, hi, n):
    """n whole numbers spread evenly over lo..hi (one: the middle)."""
    return np.array([(lo + hi + 1) // 2]) if n == 1 else np.linspace(lo, hi, n).round().astype(np.int64)


def _sizes(case):
    """Rows of each group, in no particular order."""
    g, each = case["groups"], case["each"]
    if not case["ragged"]:
        return np.full(g, each, dtype=np.int64)
    return _even(0, 2 * each, g) if g > 1 else np.array([each])


def _lengths(case):
    return _even(case["prefix_lo"], case["prefix"], case["groups"]), _even(case["tail_lo"], case["tail"], int(_sizes(case).sum()))


def _randn(gen, shape, dtype):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=gen)


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def _scattered(host, rows_pages, pages):
    """A table of the rows' pages, taken from a pool in no particular order; -1 behind a row's last page."""
    width = max(1, int(rows_pages.max()) if len(rows_pages) else 1)
    table = np.full((len(rows_pages), width), -1, dtype=np.int64)
    table[np.arange(width)[None] < rows_pages[:, None]] = host.permutation(pages)[: int(rows_pages.sum())]
    return table


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    host = np.random.RandomState(seed % (1 << 31))
    op = case["op"]
    if op == "attend":
        dt = DTYPES[case["dtype"]]
        hk, d, page = case["kv_heads"], case["dim"], case["page"]
        sizes = host.permutation(_sizes(case))
        active = int(sizes.sum())
        rows = active + case["pad"]
        lens, tails = (host.permutation(x) for x in _lengths(case))
        tails = np.concatenate([tails, np.full(case["pad"], 1)]) if case["pad"] else tails
        need = -(-tails // page)
        pages = max(1, int(need.sum()))
        table = _scattered(host, need, pages)
        s = max(1, case["prefix"])
        state = dict(q=_randn(gen, (rows, case["heads"], d), dt), k=_randn(gen, (case["groups"], s, hk, d), dt),
                     v=_randn(gen, (case["groups"], s, hk, d), dt), k_pages=_randn(gen, (pages, page, hk, d), dt),
                     v_pages=_randn(gen, (pages, page, hk, d), dt), lens=_i32(lens), tails=_i32(tails), table=_i32(table),
                     offsets=_i32(np.concatenate([[0], np.cumsum(sizes)])), active=active, most=int(sizes.max()),
                     out=torch.zeros(rows, case["heads"], d, dtype=dt, device="cuda"))
        # the norms on queries and keys of the decoders that use this leave them of unit scale, times a learned weight
        state["q"] *= 1.5
    elif op in ("fork", "compact"):
        page = case["page"]
        if op == "fork":
            lens = host.permutation(_even(case["lo"], case["hi"], case["parents"]))
            need = -(-lens // page)
            pages = int(need.sum()) + case["children"] + 5
            rows = case["parents"] + case["children"]
            table = np.full((rows, max(1, -(-case["hi"] // page))), -1, dtype=np.int64)
            used = _scattered(host, need, pages)
            table[: case["parents"], : used.shape[1]] = used
            lens = np.concatenate([lens, np.zeros(case["children"], dtype=np.int64)])
        else:
            pages = case["pages"]
            used = max(1, pages * case["live"] // 100)
            rows = min(case["rows"], used)
            need = _even(1, 2 * (used // rows) - 1, rows)
            need = np.minimum(need, 1 + (used - rows) // rows * 2)
            while need.sum() > used:
                need[np.argmax(need)] -= 1
            need = host.permutation(need)
            table = _scattered(host, need, pages)
            lens = need * page - host.randint(0, page, rows)
        refs = np.bincount(table[table >= 0], minlength=pages)
        shape = (case["layers"], pages, page, case["kv_heads"], case["dim"])
        state = dict(k=_randn(gen, shape, torch.bfloat16), v=_randn(gen, shape, torch.bfloat16), table=_i32(table),
                     lens=_i32(lens), refs=_i32(refs))
        if op == "fork":
            state["src"] = _i32(host.randint(0, case["parents"], case["children"]))
            state["dst"] = _i32(case["parents"] + host.permutation(case["children"]))
        else:
            state["saved"] = (state["table"].clone(), state["refs"].clone())
    elif op == "start":
        page, rows, count = case["page"], case["rows"], case["count"]
        width = -(-count // page)
        held = host.randint(0, width + 1, rows)  # pages that the last batch still has
        table = np.full((rows, width), -1, dtype=np.int64)
        table[np.arange(width)[None] < held[:, None]] = host.permutation(case["pages"])[: int(held.sum())]
        refs = np.bincount(table[table >= 0], minlength=case["pages"])
        # pages that another user of the pool holds
        refs[host.permutation(np.flatnonzero(refs == 0))[: max(0, case["pages"] - rows * width)]] = 1
        kv = torch.zeros(1, case["pages"], page, 1, 64, dtype=torch.bfloat16, device="cuda")
        state = dict(k=kv, v=kv.clone(), table=_i32(table), lens=_i32(held * page), refs=_i32(refs))
    else:
        b, v, t = case["rows"], case["vocab"], case["tokens"]
        logits = torch.empty(b, v, device="cuda").normal_(0.0, 4.0, generator=gen).to(DTYPES[case["dtype"]])
        # tokens as decoders repeat them: often the low ids, now and then any
        u = torch.rand(b, t, device="cuda", generator=gen, dtype=torch.float64)
        state = dict(logits=logits, history=(u.pow(3) * v).long().clamp(max=v - 1),
                     hlens=_i32(host.permutation(_even(0, t, b))),
                     repetition=torch.rand(b, device="cuda", generator=gen) * 0.5 + 1.0,
                     presence=torch.rand(b, device="cuda", generator=gen), frequency=torch.rand(b, device="cuda", generator=gen) * 0.2,
                     bias=None, mask=None, state=None, out=torch.empty_like(logits))
        if case["bias"]:
            state["bias"] = torch.randn(v, device="cuda", generator=gen)
        if case["mask"]:
            words = -(-v // 32)
            state["mask"] = torch.randint(-(1 << 31), 1 << 31, (case["mask"], words), device="cuda", generator=gen).to(torch.int32)
            state["state"] = _i32(host.randint(0, case["mask"], b))
    state["case"] = dict(case)
    return state


# ------------------------------------------------------------------------------------------------------ one pass
def run(state):
    return {"attend": _run_attend, "fork": _run_fork, "compact": _run_compact, "start": _run_start,
            "penal": _run_penal}[state["case"]["op"]](state)


def _run_attend(s):
    if own:
        from viktor_b200.ops import shared_prefix_attention
        out, lse = shared_prefix_attention(s["q"], s["k"], s["v"], s["lens"], s["offsets"], s["k_pages"], s["v_pages"],
                                           s["table"], s["tails"], out=s["out"], return_lse=True)
        return {"out": out, "lse": lse[: s["active"]]}
    n, hk = s["active"], s["k"].shape[2]
    h, d = s["q"].shape[1:]
    r, groups, most = h // hk, s["k"].shape[0], s["most"]
    q = s["q"][:n].float().reshape(n, hk, r, d)
    rows = torch.arange(n, device="cuda")
    group = torch.searchsorted(s["offsets"][1:].long(), rows, right=True)
    place = rows - s["offsets"].long()[group]
    # prefixes: the rows of a group side by side, one product for each group and KV head
    qg = torch.zeros(groups, most, hk, r, d, device="cuda")
    qg[group, place] = q
    qg = qg.permute(0, 2, 1, 3, 4).reshape(groups, hk, most * r, d)
    scale = d ** -0.5
    sp = (qg @ s["k"].float().permute(0, 2, 3, 1)).mul_(scale)
    sp.masked_fill_((torch.arange(s["k"].shape[1], device="cuda") >= s["lens"][:, None])[:, None, None], -INF)
    # tails: every row's pages laid out one after another
    t = s["table"][:n].clamp(min=0).long()
    kt, vt = (x[t].reshape(n, -1, hk, d).float() for x in (s["k_pages"], s["v_pages"]))
    st = (q @ kt.permute(0, 2, 3, 1)).mul_(scale)
    st.masked_fill_((torch.arange(kt.shape[1], device="cuda") >= s["tails"][:n, None])[:, None, None], -INF)
    # one softmax over both
    mp = sp.amax(-1).reshape(groups, hk, most, r).transpose(1, 2)
    m = torch.maximum(mp[group, place], st.amax(-1))
    m = torch.where(m == -INF, 0.0, m)
    mg = torch.zeros(groups, most, hk, r, device="cuda")
    mg[group, place] = m
    sp.sub_(mg.transpose(1, 2).reshape(groups, hk, most * r, 1)).exp_()
    st.sub_(m[..., None]).exp_()
    lp = sp.sum(-1).reshape(groups, hk, most, r).transpose(1, 2)[group, place]
    op = (sp @ s["v"].float().permute(0, 2, 1, 3)).reshape(groups, hk, most, r, d).transpose(1, 2)[group, place]
    lsum = lp + st.sum(-1)
    o = (op + st @ vt.permute(0, 2, 1, 3)) / torch.where(lsum == 0, 1.0, lsum)[..., None]
    s["out"][:n] = o.reshape(n, h, d).to(s["out"].dtype)
    return {"out": s["out"], "lse": (m + lsum.log()).reshape(n, h)}


def _pages(s):
    if "pages" not in s:
        from viktor_b200.ops import KVPages
        s["pages"] = KVPages(s["k"], s["v"], s["table"], s["lens"], s["refs"])
    return s["pages"]


def _bookkeeping(s, data=True):
    got = {k: s[k] for k in ("table", "lens", "refs")}
    return {**got, "k": s["k"], "v": s["v"]} if data else got


def _plain_free(s, rows):
    old = s["table"][rows]
    s["refs"].index_add_(0, old.clamp(min=0).reshape(-1), -(old >= 0).reshape(-1).int())
    s["table"][rows] = -1
    s["lens"][rows] = 0


def _run_fork(s):
    """The children of the last pass are given up, then made anew."""
    if own:
        from viktor_b200.ops import pages_fork, pages_free
        pages = _pages(s)
        pages_free(pages, s["dst"])
        pages_fork(pages, s["src"], s["dst"])
        return _bookkeeping(s)
    src, dst, page, width = s["src"].long(), s["dst"].long(), s["k"].shape[2], s["table"].shape[1]
    _plain_free(s, dst)
    lens = s["lens"][src].long()
    full, part = lens // page, lens % page
    free = torch.argsort((s["refs"] > 0).int(), stable=True)  # free pages first, the lowest first
    wants = part > 0
    fresh = free[(torch.cumsum(wants, 0) - 1).clamp(min=0)]
    col = torch.arange(width, device="cuda")
    shared = torch.where(col < full[:, None], s["table"][src], -1)
    s["refs"].index_add_(0, shared.clamp(min=0).reshape(-1), (shared >= 0).reshape(-1).int())
    s["refs"].index_add_(0, fresh, wants.int())
    s["table"][dst] = torch.where((col == full[:, None]) & wants[:, None], fresh.int()[:, None], shared)
    s["lens"][dst] = lens.int()
    # the partial pages; where there is none, a page in use is written onto itself
    last = s["table"][src, full.clamp(max=width - 1)].long()
    last, to = torch.where(wants, last, free[-1]), torch.where(wants, fresh, free[-1])
    keep = (torch.arange(page, device="cuda") < part[:, None]) | ~wants[:, None]
    for x in (s["k"], s["v"]):
        x[:, to] = torch.where(keep[None, :, :, None, None], x[:, last], x[:, to])
    return _bookkeeping(s)


def _run_compact(s):
    """The bookkeeping of a pool is loaded as it was kept, and its pages are compacted."""
    s["table"].copy_(s["saved"][0])
    s["refs"].copy_(s["saved"][1])
    if own:
        from viktor_b200.ops import pages_compact
        return {**_bookkeeping(s), "live": pages_compact(_pages(s))}
    used = s["refs"] > 0
    live = used.sum()
    at = torch.arange(used.numel(), device="cuda")
    holes, movers = ~used & (at < live), used & (at >= live)
    most = used.numel() // 2
    to = torch.argsort((~holes).int(), stable=True)[:most]
    of = torch.argsort((~movers).int(), stable=True)[:most]
    moves = at[:most] < movers.sum()
    goes = at.clone()
    goes[of] = torch.where(moves, to, of)
    for x in (s["k"], s["v"]):
        x[:, to] = torch.where(moves[None, :, None, None, None], x[:, of], x[:, to])
    old = s["table"]
    s["table"].copy_(torch.where(old >= 0, goes[old.clamp(min=0).long()].int(), old))
    refs = torch.zeros_like(s["refs"])
    refs.index_add_(0, goes, torch.where(used, s["refs"], 0))
    s["refs"].copy_(refs)
    return {**_bookkeeping(s), "live": live.int().reshape(1)}


def _run_start(s):
    """The rows of the last batch are given up and each gets room for its new tokens."""
    count = s["case"]["count"]
    if own:
        from viktor_b200.ops import pages_extend, pages_free
        pages = _pages(s)
        pages_free(pages)
        page, slot = pages_extend(pages, count)
        return {**_bookkeeping(s, False), "page": page, "slot": slot}
    rows, width = s["table"].shape
    _plain_free(s, torch.arange(rows, device="cuda"))
    free = torch.argsort((s["refs"] > 0).int(), stable=True)[: rows * width].reshape(rows, width)
    s["refs"].index_add_(0, free.reshape(-1), torch.ones(rows * width, dtype=torch.int32, device="cuda"))
    s["table"].copy_(free)
    s["lens"].fill_(count)
    at = torch.arange(count, device="cuda")
    size = s["k"].shape[2]
    return {**_bookkeeping(s, False), "page": s["table"][:, at // size], "slot": (at % size).int().expand(rows, count)}


def _run_penal(s):
    if own:
        from viktor_b200.ops import penalize_logits
        return penalize_logits(s["logits"], s["history"], s["hlens"], repetition=s["repetition"], presence=s["presence"],
                               frequency=s["frequency"], bias=s["bias"], mask=s["mask"], mask_index=s["state"], out=s["out"])
    x = s["logits"].float()
    b, v = x.shape
    counts = torch.zeros(b, v, device="cuda")
    counts.scatter_add_(1, s["history"], (torch.arange(s["history"].shape[1], device="cuda") < s["hlens"][:, None]).float())
    rep = s["repetition"][:, None]
    x = torch.where(counts > 0, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][:, None] * counts - s["presence"][:, None] * (counts > 0)
    if s["bias"] is not None:
        x = x + s["bias"]
    if s["mask"] is not None:
        at = torch.arange(v, device="cuda")
        allowed = (s["mask"][:, at // 32] >> (at % 32).int()) & 1
        x = x.masked_fill(allowed[s["state"].long()] == 0, -INF)
    s["out"].copy_(x)
    return s["out"]


# ------------------------------------------------------------------------------------------------------ floors
def work(case):
    op = case["op"]
    if op == "attend":
        sizes, (lens, tails) = np.sort(_sizes(case)), _lengths(case)
        rows, row = int(sizes.sum()), case["kv_heads"] * case["dim"] * 2
        # which group has which prefix is the seed's: the mean stands for it
        read = 2 * row * (int(lens.sum()) + int(tails.sum())) + rows * case["heads"] * case["dim"] * 2
        wide = rows * float(lens.mean()) + int(tails.sum())
        return {"bytes": int(read + rows * case["heads"] * (case["dim"] * 2 + 4)), "flops": int(4 * case["heads"] * case["dim"] * wide)}
    if op == "fork":
        lens, page = _even(case["lo"], case["hi"], case["parents"]), case["page"]
        part, each = float((lens % page).mean()), float((-(-lens // page)).mean())
        copied = case["children"] * part * case["layers"] * 2 * case["kv_heads"] * case["dim"] * 2
        return {"bytes": int(2 * copied + case["children"] * (8 * each + 12)), "flops": 0}
    if op == "compact":
        used = case["pages"] * case["live"] // 100
        moves = used * (case["pages"] - used) / case["pages"]
        size = case["layers"] * 2 * case["page"] * case["kv_heads"] * case["dim"] * 2
        return {"bytes": int(2 * moves * size + 8 * case["pages"] + 8 * used), "flops": 0}
    if op == "start":
        cells = case["rows"] * -(-case["count"] // case["page"])
        return {"bytes": int(8 * cells + 8 * case["pages"] + 8 * case["rows"] * case["count"]), "flops": 0}
    size = 4 if case["dtype"] == "f32" else 2
    tokens = int(_even(0, case["tokens"], case["rows"]).sum())
    cells = case["rows"] * case["vocab"]
    masks = min(case["mask"], case["rows"]) * case["vocab"] // 8
    return {"bytes": 2 * size * cells + 8 * tokens + masks + 4 * case["vocab"] * case["bias"], "flops": 4 * cells}


# ------------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attend":
        return _exact_attend(s)
    if case["op"] == "penal":
        return _exact_penal(s)
    return None  # whole numbers and copies


def _exact_attend(s):
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full((s["active"], s["q"].shape[1]), -INF, dtype=torch.float64, device="cuda")
    off, lens, tails = s["offsets"].tolist(), s["lens"].tolist(), s["tails"].tolist()
    heads, d = s["q"].shape[1:]
    hk = s["k"].shape[2]
    for g in range(len(lens)):
        kp, vp = (x[g, : lens[g]].double() for x in (s["k"], s["v"]))
        for b in range(off[g], off[g + 1]):
            n = tails[b]
            pages = s["table"][b, : -(-n // s["k_pages"].shape[1])].long()
            k, v = (torch.cat([a, x[pages].flatten(0, 1)[:n].double()]) for a, x in ((kp, s["k_pages"]), (vp, s["v_pages"])))
            if k.shape[0]:
                q = s["q"][b].double().view(hk, heads // hk, d)
                z = torch.einsum("hrd,nhd->hrn", q, k) / math.sqrt(d)
                out[b] = torch.einsum("hrn,nhd->hrd", torch.softmax(z, -1), v).reshape(heads, d)
                lse[b] = torch.logsumexp(z, -1).reshape(heads)
    return {"out": out, "lse": lse}


def _exact_penal(s):
    x = s["logits"].double()
    rows = []
    for b, n in enumerate(s["hlens"].tolist()):
        c = torch.bincount(s["history"][b, :n], minlength=x.shape[1]).double()
        seen, rep = c > 0, s["repetition"][b].double()
        y = x[b] * torch.where(seen, torch.where(x[b] > 0, 1 / rep, rep), 1.0)
        y = y - c * s["frequency"][b].double() - seen * s["presence"][b].double()
        if s["bias"] is not None:
            y = y + s["bias"].double()
        if s["mask"] is not None:
            words = s["mask"][s["state"][b]].long() & 0xFFFFFFFF
            bits = (words[:, None] >> torch.arange(32, device="cuda")) & 1
            y[bits.flatten()[: y.numel()] == 0] = -INF
        rows.append(y)
    return torch.stack(rows)
