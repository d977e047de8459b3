"""The operators of the paged Q4_0 key-value cache: what is timed and compared.

A case names its operator (`kind`) and its sizes:

  plan    block tables and slot maps from the requests' lengths: every entry
          takes n_new more positions, then gives them back (a draft that was
          rejected, a request that ended)
  append  K and V rows into their slots, then the slots read out again
  decode  attention of one token per entry over its pages
  step    the same with the token's own K and V appended in the call, then the
          new slots read out
  attend  ragged query rows over their entries' pages: prompt chunks (causal)
          or cross attention to an encoder's states

The cache holds ggml Q4_0 blocks of 32 elements; the plain form keeps them as
codes and scales, and every output that is held in them is returned as the
values they stand for.  Slot s of the cache is position s % page of page
s // page.  The entries' lengths are spread evenly over their range and dealt
out by the seed; pages are dealt out at random, as in a pool in use.
"""
import math

import numpy as np
import torch

own = False


def listed():
    return [
        # a server's 48 sessions grow by their next token: the smallest plan
        {"name": "plan, a token each", "kind": "plan", "entries": 48, "page": 64, "longest": 3000, "new": 1,
         "spare": 1.5},
        # 256 requests, half of them with prompts, into a pool that just holds them
        {"name": "plan, prompts", "kind": "plan", "entries": 256, "page": 16, "longest": 8192, "new": 4096,
         "spare": 1.0},
        # the K and V of 48 sessions' tokens, views of the packed QKV rows
        {"name": "append, a token each", "kind": "append", "entries": 48, "rows": 1, "heads": 32, "kv": 32, "dim": 128,
         "page": 64, "type": "float32"},
        # six prompts, 32 query heads over 8 kv heads, in 16 bits
        {"name": "append, prompts", "kind": "append", "entries": 6, "rows": 1500, "heads": 32, "kv": 8, "dim": 128,
         "page": 128, "type": "bfloat16"},
        # one user's token: latency
        {"name": "decode, one session", "kind": "decode", "entries": 1, "heads": 32, "kv": 32, "dim": 128, "page": 64,
         "shortest": 700, "longest": 700, "window": 0, "type": "float32"},
        # 64 sessions of the temporal transformer at every age of its 3000 positions
        {"name": "decode, 64 sessions", "kind": "decode", "entries": 64, "heads": 32, "kv": 32, "dim": 128, "page": 64,
         "shortest": 100, "longest": 3000, "window": 0, "type": "float32"},
        # long contexts, 4 query heads to a kv head, few entries: the split
        {"name": "decode, long, grouped", "kind": "decode", "entries": 12, "heads": 32, "kv": 8, "dim": 128,
         "page": 128, "shortest": 2000, "longest": 32000, "window": 0, "type": "bfloat16"},
        # 40 sessions of a small model, one token with its append
        {"name": "step, 64-wide heads", "kind": "step", "entries": 40, "heads": 16, "kv": 16, "dim": 64, "page": 32,
         "shortest": 5, "longest": 1000, "window": 0, "type": "float32"},
        # 256 sessions that see the last 512 positions of longer histories
        {"name": "step, window", "kind": "step", "entries": 256, "heads": 32, "kv": 8, "dim": 128, "page": 64,
         "shortest": 40, "longest": 4000, "window": 512, "type": "bfloat16"},
        # the next piece of one prompt: latency
        {"name": "attend, a short chunk", "kind": "attend", "entries": 1, "heads": 32, "kv": 32, "dim": 128, "page": 64,
         "few": 37, "rows": 37, "shortest": 500, "longest": 500, "causal": True, "window": 0, "type": "bfloat16"},
        # eight prompts in chunks of up to 1024 tokens: the largest product
        {"name": "attend, prompts", "kind": "attend", "entries": 8, "heads": 32, "kv": 8, "dim": 128, "page": 128,
         "few": 200, "rows": 1024, "shortest": 300, "longest": 4000, "causal": True, "window": 0, "type": "bfloat16"},
        # a decoder's few rows against 12 encoders' 1500 states
        {"name": "attend, cross", "kind": "attend", "entries": 12, "heads": 16, "kv": 16, "dim": 64, "page": 32,
         "few": 1, "rows": 24, "shortest": 200, "longest": 1500, "causal": False, "window": 0, "type": "float16"},
    ]


def _log_int(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        c = _draw(rng)
        w = work(c)
        if w["bytes"] <= 4.5e8 and w["flops"] <= 2.4e11 and _room(c):  # within the largest listed
            return c


def _room(c):
    """Whether a drawn case's cache and scores, all in 32 bits, are no larger than the listed ones'."""
    if c["kind"] in ("plan", "append"):
        return True
    long = c["longest"] + (c["rows"] if c["kind"] == "attend" else 0)
    rows = c.get("rows", 1)
    return c["entries"] * long * c["kv"] * c["dim"] <= 8e8 and c["entries"] * rows * long * c["heads"] <= 1.3e9


def _draw(rng):
    kind = rng.choice(["plan", "append", "decode", "decode", "step", "step", "attend", "attend", "attend"])
    if kind == "plan":
        page = rng.choice([16, 32, 64, 128, 256])
        return {"kind": kind, "entries": _log_int(rng, 1, 1024), "page": page, "longest": _log_int(rng, 100, 20000),
                "new": rng.choice([1, rng.randint(2, 9), _log_int(rng, 10, 4096)]),
                "spare": rng.choice([1.0, 1.2, 2.0])}
    dim = rng.choice([64, 128, 128])
    kv = rng.choice([1, 2, 4, 8, 8, 16, 20, 32])
    heads = kv * rng.choice([1, 1, 2, 3, 4, 8, 16])
    heads = heads if heads <= 64 else kv
    page = rng.choice([32, 64, 128, 256] if dim == 64 else [16, 32, 64, 128, 256])
    c = {"kind": kind, "entries": 0, "heads": heads, "kv": kv, "dim": dim, "page": page}
    if kind == "append":
        c.update(entries=_log_int(rng, 1, 200), rows=_log_int(rng, 1, 3000),
                 type=rng.choice(["float32", "float16", "bfloat16"]))
        return c
    longest = _log_int(rng, 1, 40000)
    c.update(entries=_log_int(rng, 1, 256), shortest=rng.choice([0, max(1, longest // 20), longest]), longest=longest,
             window=rng.choice([0, 0, _log_int(rng, 1, 3000)]), type=rng.choice(["float32", "float16", "bfloat16"]))
    if kind == "step":
        c["shortest"] = max(1, c["shortest"])
    if kind == "attend":
        rows = _log_int(rng, 1, 1500)
        c.update(entries=_log_int(rng, 1, 24), few=rng.choice([0, 1, rows]), rows=rows,
                 causal=rng.random() < 0.6, type=rng.choice(["float16", "bfloat16"]))
        c["longest"] = min(6000, c["longest"])
        c["shortest"] = min(c["shortest"], c["longest"])
        if not c["causal"]:
            c["window"] = 0
    return c


# ---- sizes of a case -------------------------------------------------------


def _spread(lo, hi, n):
    """n whole numbers of [lo, hi], evenly spread."""
    return [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _sizes(c, seed=None):
    """An attention case's lengths and rows per entry, dealt out by the seed."""
    n = c["entries"]
    lens = _spread(c["shortest"], c["longest"], n)
    rows = _spread(c["few"], c["rows"], n) if c["kind"] == "attend" else [1] * n
    if c["kind"] == "attend" and c["causal"]:  # the rows are positions too
        lens = [a + b for a, b in zip(lens, rows)]
    if seed is not None:
        order = np.random.default_rng([seed, 1]).permutation(n)
        lens, rows = [lens[i] for i in order], [rows[i] for i in order]
    return lens, rows


def _plan_sizes(c, seed=0):
    """A plan case's lengths and new positions per entry, dealt out by the seed."""
    r = np.random.default_rng([seed, 2])
    n = c["entries"]
    new = np.ones(n, dtype=np.int64)
    if c["new"] > 1:  # every second entry has a prompt, one in eight has nothing
        i = np.arange(n)
        prompt = np.exp(np.array(_spread(0, 1000, n)) / 1000.0 * math.log(c["new"])).astype(np.int64)
        new = np.where(i % 8 == 7, 0, np.where(i % 2 == 0, prompt, 1))
    return np.array(_spread(0, c["longest"], n))[r.permutation(n)], new[r.permutation(n)]


def _visible(c, n_rows, length, row):
    """How many positions a row of an entry sees."""
    last = length - n_rows + row + 1 if c.get("causal", True) else length
    return max(0, min(last, c["window"]) if c["window"] else last)


def _itemsize(c):
    return 4 if c["type"] == "float32" else 2


def work(c):
    if c["kind"] == "plan":
        new = _plan_sizes(c)[1]
        # lengths, requests, starts and states twice; a token's slot, position and
        # entry; a page's place in the list and in the table, there and back
        return {"bytes": 4.0 * (8 * len(new) + 3 * int(new.sum()) + 4 * int((new // c["page"]).sum())), "flops": 0.0}
    block = c["kv"] * c["dim"] // 32 * 18
    if c["kind"] == "append":
        n = sum(_spread(max(1, c["rows"] // 4), c["rows"], c["entries"]))
        return {"bytes": float(n * 2 * (c["kv"] * c["dim"] * (_itemsize(c) + 4) + 2 * block)), "flops": 0.0}
    lens, rows = _sizes(c)
    total = seen = 0
    for length, n in zip(lens, rows):
        if n:
            total += _visible(dict(c, causal=False), n, length, 0) if c["kind"] != "attend" else \
                min(length, c["window"] + n - 1) if c["window"] else length
            if not c.get("causal", True):
                seen += n * length
            elif c["window"]:
                seen += sum(_visible(c, n, length, i) for i in range(n))
            else:
                seen += n * (length - n) + n * (n + 1) // 2
    size = _itemsize(c)
    b = total * 2 * block + sum(rows) * c["heads"] * c["dim"] * 2 * size
    if c["kind"] == "step":
        b += c["entries"] * 2 * (c["kv"] * c["dim"] * (size + 4) + block)
    return {"bytes": float(b), "flops": 4.0 * seen * c["heads"] * c["dim"]}


# ---- prepare ---------------------------------------------------------------


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed & (2**62 - 1))
    return g


def _kv(g, *shape):
    """K or V rows: N(0, 1), one element in a hundred 8 times as large."""
    x = torch.randn(*shape, generator=g, device="cuda")
    return torch.where(torch.rand(*shape, generator=g, device="cuda") < 0.01, x * 8, x)


def _i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def _tables(lens, page, seed, extra=0):
    """A block table of the lengths (+ extra pages for each) with pages in
    random order, and the pages of the pool."""
    need = [-(-n // page) + extra for n in lens]
    width = max(1, max(need))
    ids = np.random.default_rng([seed, 4]).permutation(sum(need) + 3)
    table = np.zeros((len(lens), width), dtype=np.int64)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    return table, ids[at:], len(ids)


def _cache(c, n_pages, seed):
    """Every slot's K and V rows, from the seed."""
    g = _generator(seed * 1000003 + 1)
    n = n_pages * c["page"]
    return _kv(g, n, c["kv"], c["dim"]), _kv(g, n, c["kv"], c["dim"])


def _rows(c, n, seed):
    """n tokens' q, k and v: views of packed rows, as a QKV projection leaves them."""
    g = _generator(seed * 7 + 5)
    h, kv, d = c["heads"], c["kv"], c["dim"]
    x = torch.cat((torch.randn(n, h, d, generator=g, device="cuda"), _kv(g, n, 2 * kv, d)), dim=1)
    x = x.to(getattr(torch, c["type"]))
    return x[:, :h], x[:, h:h + kv], x[:, h + kv:]


def _pool(c, n_pages, k, v):
    """The cache with K and V rows k, v in slots 0..: the library's, or codes and scales."""
    slots = torch.arange(n_pages * c["page"], dtype=torch.int32, device="cuda")
    if own:
        from bmo_jetson_amd import KVPages
        pages = KVPages(1, n_pages, c["page"], c["kv"], c["dim"])
        pages.append(0, slots, k, v, stream=torch.cuda.current_stream())
        torch.cuda.synchronize()
        return pages
    shape = (n_pages * c["page"], c["kv"], c["dim"] // 32)
    pool = [torch.zeros(*shape, 32, dtype=torch.uint8, device="cuda") if i % 2 == 0 else
            torch.zeros(*shape, dtype=torch.float16, device="cuda") for i in range(4)]
    _store(pool, slots.long(), k, v)
    return pool


def _workspace(pool, heads):
    if own:
        return torch.empty(pool.workspace_bytes(heads), dtype=torch.uint8, device="cuda")
    return None


def prepare(case, seed):
    return globals()["_prepare_" + case["kind"]](case, seed)


def _prepare_plan(c, seed):
    lens, new = _plan_sizes(c, seed)
    page = c["page"]
    table, free, n_pages = _tables(list(lens), page, seed)
    width = -(-(c["longest"] + c["new"]) // page)
    wide = np.full((len(lens), width), -1, dtype=np.int64)
    wide[:, :table.shape[1]] = table
    more = int(int((new // page + 1).sum()) * c["spare"])  # pages for what is new
    free = np.concatenate((free, np.arange(n_pages, n_pages + more)))
    n_pages += more
    pad = np.zeros(n_pages + 2, dtype=np.int64)
    pad[0], pad[2:2 + len(free)] = len(free), free
    n = int(new.sum())
    s = {"kind": "plan", "page": page, "lens": _i32(lens), "table": _i32(wide), "free": _i32(pad), "new": _i32(new),
         "back": _i32(-new), "tokens": n, "pool": None}
    for name in ("slots", "positions", "entries"):
        s[name] = torch.full((max(1, n),), -7, dtype=torch.int32, device="cuda")
    s["start"], s["start2"] = (torch.zeros(len(lens) + 1, dtype=torch.int32, device="cuda") for _ in range(2))
    s["status"], s["status2"] = (torch.zeros(len(lens), dtype=torch.int32, device="cuda") for _ in range(2))
    if own:
        from bmo_jetson_amd import KVPages
        s["pool"] = KVPages(1, n_pages, page, 1, 64 if page % 32 == 0 else 128)
    return s


def _prepare_append(c, seed):
    rows = _spread(max(1, c["rows"] // 4), c["rows"], c["entries"])
    r = np.random.default_rng([seed, 6])
    first = [int(x) for x in r.integers(0, 3 * c["page"], c["entries"])]  # positions the entries hold already
    ends = [a + b for a, b in zip(first, rows)]
    table, _, n_pages = _tables(ends, c["page"], seed)
    slots = []
    for i, (a, b) in enumerate(zip(first, ends)):
        p = np.arange(a, b)
        slots.append(table[i, p // c["page"]] * c["page"] + p % c["page"])
    slots = np.concatenate(slots)
    slots[r.permutation(len(slots))[:len(slots) // 20]] = -1  # rows of padding
    _, k, v = _rows(c, len(slots), seed)
    old_k, old_v = _cache(c, n_pages, seed)
    out = [torch.zeros(len(slots), c["kv"], c["dim"], device="cuda") for _ in range(2)]
    return {"kind": "append", "pool": _pool(c, n_pages, old_k, old_v), "slots": _i32(slots), "k": k, "v": v, "out": out}


def _attention_state(c, seed):
    lens, rows = _sizes(c, seed)
    table, _, n_pages = _tables(lens, c["page"], seed)
    k, v = _cache(c, n_pages, seed)
    pool = _pool(c, n_pages, k, v)
    q, k, v = _rows(c, sum(rows), seed)
    return {"kind": c["kind"], "pool": pool, "lens": _i32(lens), "table": _i32(table), "q": q, "k": k, "v": v,
            "out": torch.zeros(q.shape, dtype=q.dtype, device="cuda"), "page": c["page"], "longest": max(lens),
            "window": c["window"], "work": _workspace(pool, c["heads"])}, lens, rows, table


def _prepare_decode(c, seed):
    return _attention_state(c, seed)[0]


def _prepare_step(c, seed):
    s, lens, _, table = _attention_state(c, seed)
    s["slots"] = _i32([table[i, (n - 1) // c["page"]] * c["page"] + (n - 1) % c["page"] for i, n in enumerate(lens)])
    s["new"] = [torch.zeros(len(lens), c["kv"], c["dim"], device="cuda") for _ in range(2)]
    return s


def _prepare_attend(c, seed):
    s, lens, rows, _ = _attention_state(c, seed)
    s["start"] = _i32(np.concatenate(([0], np.cumsum(rows))))
    s.update(causal=c["causal"], rows=max(rows))
    return s


# ---- run -------------------------------------------------------------------


def run(state):
    return globals()["_run_" + state["kind"]](state)


def _run_plan(s):
    if own:
        stream = torch.cuda.current_stream()
        s["pool"].plan(s["free"], s["new"], s["lens"], s["table"], s["start"], s["slots"], s["positions"], s["entries"],
                       s["status"], stream=stream)
        s["pool"].plan(s["free"], s["back"], s["lens"], s["table"], s["start2"], status=s["status2"], stream=stream)
    else:
        _plan(s, s["new"], s["tokens"], s["start"], s["status"], s["slots"], s["positions"], s["entries"])
        _plan(s, s["back"], 0, s["start2"], s["status2"])
    return {k: s[k] for k in ("start", "slots", "positions", "entries", "status", "status2", "lens", "table", "free")}


def _run_append(s):
    if own:
        stream = torch.cuda.current_stream()
        s["pool"].append(0, s["slots"], s["k"], s["v"], stream=stream)
        s["pool"].gather(0, s["slots"], *s["out"], stream=stream)
        return {"k": s["out"][0], "v": s["out"][1]}
    slots = s["slots"].long()
    real = slots >= 0
    _store(s["pool"], slots[real], s["k"][real], s["v"][real])
    k, v = _load(s["pool"], slots.clamp(min=0))
    return {"k": torch.where(real[:, None, None], k, 0.0), "v": torch.where(real[:, None, None], v, 0.0)}


def _run_decode(s):
    if own:
        s["pool"].decode(0, s["lens"], s["table"], s["q"], s["out"], window=s["window"], max_len=s["longest"],
                         workspace=s["work"], stream=torch.cuda.current_stream())
        return {"out": s["out"]}
    n = torch.ones_like(s["lens"])
    return {"out": _attention(s, s["q"][:, None], n, True)[:, 0].to(s["q"].dtype)}


def _run_step(s):
    if own:
        stream = torch.cuda.current_stream()
        s["pool"].append_decode(0, s["lens"], s["table"], s["q"], s["k"], s["v"], s["out"], window=s["window"],
                                max_len=s["longest"], workspace=s["work"], stream=stream)
        s["pool"].gather(0, s["slots"], *s["new"], stream=stream)
        return {"out": s["out"], "k": s["new"][0], "v": s["new"][1]}
    slots = s["slots"].long()
    _store(s["pool"], slots, s["k"], s["v"])
    k, v = _load(s["pool"], slots)
    n = torch.ones_like(s["lens"])
    return {"out": _attention(s, s["q"][:, None], n, True)[:, 0].to(s["q"].dtype), "k": k, "v": v}


def _run_attend(s):
    if own:
        s["pool"].attend(0, s["start"], s["lens"], s["table"], s["q"], s["out"], causal=s["causal"], window=s["window"],
                         max_rows=s["rows"], max_len=s["longest"], workspace=s["work"],
                         stream=torch.cuda.current_stream())
        return {"out": s["out"]}
    start, total = s["start"].long(), s["q"].shape[0]
    n = start[1:] - start[:-1]
    entry = torch.repeat_interleave(torch.arange(n.numel(), device="cuda"), n, output_size=total)
    row = torch.arange(total, device="cuda") - start[entry]
    q = torch.zeros(n.numel(), max(1, s["rows"]), *s["q"].shape[1:], device="cuda")
    q[entry, row] = s["q"].float()
    return {"out": _attention(s, q, n, s["causal"])[entry, row].to(s["q"].dtype)}


# ---- the plain forms -------------------------------------------------------


def _plan(s, n_new, tokens, start, status, slots=None, positions=None, entries=None):
    page, (n, width) = s["page"], s["table"].shape
    lens, table, free = s["lens"].long(), s["table"].long(), s["free"].long()
    asked = n_new.long()
    new = (lens + asked).clamp(min=0)
    count = asked.clamp(min=0)
    first = torch.cumsum(count, 0) - count
    start[:n] = first.int()
    start[n:] = (first[-1:] + count[-1:]).int()
    bad = (lens < 0) | (lens > width * page) | (new > width * page) | (first + count > tokens)
    have, want = (lens + page - 1) // page, (new + page - 1) // page
    need = torch.where(~bad & (asked > 0), want - have, 0)
    upto = torch.cumsum(need, 0)
    short = (need > 0) & (upto > free[0])
    good = ~bad & ~short
    status.copy_(torch.where(bad, 2, torch.where(short, 1, 0)))
    given = torch.where(good, need, 0)
    column = torch.arange(width, device="cuda")[None, :]
    # pages taken from the end of the list
    take = good[:, None] & (column >= have[:, None]) & (column < want[:, None])
    at = free[0] - 1 - (upto - need)[:, None] - (column - have[:, None])
    table = torch.where(take, free[2 + at.clamp(0, free.numel() - 3)], table)
    left = free[0] - given.sum()
    # pages put back, the last one first
    back = torch.where(good & (asked < 0), have - want, 0)
    before = torch.cumsum(back, 0) - back
    gone = (back > 0)[:, None] & (column >= want[:, None]) & (column < have[:, None])
    at = left + back.sum() - 1 - before[:, None] - (column - want[:, None])
    spill = torch.cat((free, free[:1]))  # one place more, for what is not put back
    spill = spill.scatter(0, torch.where(gone, 2 + at, free.numel()).reshape(-1), table.reshape(-1))
    free = spill[:-1]
    free[:1] = left + back.sum()
    s["free"].copy_(free)
    s["table"].copy_(table)
    s["lens"].copy_(torch.where(good, new, lens))
    if tokens:
        entry = torch.repeat_interleave(torch.arange(n, device="cuda"), count, output_size=tokens)
        pos = lens[entry] + torch.arange(tokens, device="cuda") - first[entry]
        slot = table[entry, (pos // page).clamp(0, width - 1)] * page + pos % page
        slots.copy_(torch.where(good[entry], slot, -1))
        positions.copy_(torch.where(good[entry], pos, -1))
        entries.copy_(entry)


def _quantize(x):
    """ggml Q4_0 of x's blocks of 32: codes 0..15 and fp16 scales."""
    b = x.float().reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    first = b.abs().argmax(dim=-1, keepdim=True)
    d = b.gather(-1, first) / -8.0
    inv = torch.where(d != 0, 1.0 / d, 0.0)
    code = (b * inv + 8.5).to(torch.int32).clamp(max=15).to(torch.uint8)
    return code, d[..., 0].to(torch.float16)


def _store(pool, slots, k, v):
    pool[0][slots], pool[1][slots] = _quantize(k)
    pool[2][slots], pool[3][slots] = _quantize(v)


def _values(code, d):
    x = (code.float() - 8.0) * d.float()[..., None]
    return x.reshape(*x.shape[:-2], x.shape[-2] * 32)


def _load(pool, slots):
    return _values(pool[0][slots], pool[1][slots]), _values(pool[2][slots], pool[3][slots])


def _attention(s, q, n, causal):
    """softmax(q k / sqrt(dim)) v of padded rows q [entries][rows][heads][dim],
    n of them an entry's, over the entries' pages."""
    page, longest = s["page"], s["longest"]
    entries, rows, heads, dim = q.shape
    slots = (s["table"].long()[:, :, None] * page + torch.arange(page, device="cuda")).reshape(entries, -1)[:, :longest]
    k, v = _load(s["pool"], slots)  # [entries][positions][kv][dim]
    kv, keys = k.shape[2], k.shape[1]
    q = q.float().reshape(entries, rows, kv, heads // kv, dim).permute(0, 2, 3, 1, 4).reshape(entries, kv, -1, dim)
    score = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()) / math.sqrt(dim)
    score = score.reshape(entries, kv, heads // kv, rows, keys)
    at = torch.arange(keys, device="cuda")[None, None, :]
    lens = s["lens"].long()[:, None, None]
    last = lens - n.long()[:, None, None] + torch.arange(rows, device="cuda")[None, :, None] if causal else lens - 1
    hide = (at > last) | (at >= lens)
    if s["window"]:
        hide = hide | (at <= last - s["window"])
    score = score.masked_fill(hide[:, None, None], -math.inf)
    top = score.amax(dim=-1, keepdim=True).clamp(min=-3e38) if keys else score
    p = torch.exp(score - top)
    total = p.sum(dim=-1, keepdim=True)
    p = torch.where(total > 0, p / total, 0.0)
    o = torch.matmul(p.reshape(entries, kv, -1, keys), v.permute(0, 2, 1, 3).contiguous())
    return o.reshape(entries, kv, heads // kv, rows, dim).permute(0, 3, 1, 2, 4).reshape(entries, rows, heads, dim)


# ---- in 64 bits ------------------------------------------------------------


def _q4_0(x):
    """The values that rows x have as Q4_0, in 64 bits: ggml's steps, each
    rounded to 32 bits on its own (the definition of the codes)."""
    b = x.float().reshape(-1, 32)
    hi, lo = b.amax(dim=1), b.amin(dim=1)
    big = torch.maximum(hi, -lo)
    place = torch.arange(32, device=b.device).expand_as(b)
    at = torch.where(b.abs() == big[:, None], place, 32).amin(dim=1)
    d = torch.div(b[torch.arange(b.shape[0], device=b.device), at], -8.0)
    inv = torch.reciprocal(d).masked_fill(d == 0, 0.0)
    code = torch.floor(torch.add(torch.mul(b, inv[:, None]), 8.5)).clamp(max=15.0)
    return ((code.double() - 8.0) * d.half().double()[:, None]).reshape(x.shape)


def exact(case, seed):
    return globals()["_exact_" + case["kind"]](case, seed)


def _exact_plan(c, seed):
    return None  # whole numbers


def _exact_append(c, seed):
    s = _prepare_slots(c, seed)
    _, k, v = _rows(c, len(s), seed)
    gone = torch.tensor(s < 0, device="cuda")[:, None, None]
    return {"k": _q4_0(k).masked_fill(gone, 0.0), "v": _q4_0(v).masked_fill(gone, 0.0)}


def _prepare_slots(c, seed):
    """The slots of an append case: which rows are padding."""
    n = sum(_spread(max(1, c["rows"] // 4), c["rows"], c["entries"]))
    r = np.random.default_rng([seed, 6])
    r.integers(0, 3 * c["page"], c["entries"])
    slots = np.zeros(n, dtype=np.int64)
    slots[r.permutation(n)[:n // 20]] = -1
    return slots


def _exact_rows(c, seed, new):
    """Each entry's attention in 64 bits, one entry after another."""
    lens, rows = _sizes(c, seed)
    table, _, n_pages = _tables(lens, c["page"], seed)
    all_k, all_v = _cache(c, n_pages, seed)
    q, new_k, new_v = _rows(c, sum(rows), seed)
    out, at = [], 0
    group = c["heads"] // c["kv"]
    for i, (length, n) in enumerate(zip(lens, rows)):
        pos = np.arange(length)
        slot = torch.tensor(table[i, pos // c["page"]] * c["page"] + pos % c["page"], device="cuda")
        k, v = all_k[slot], all_v[slot]
        if new:
            k[length - 1], v[length - 1] = new_k[i].float(), new_v[i].float()
        k, v = _q4_0(k), _q4_0(v)
        x = q[at:at + n].double()
        at += n
        y = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
        if length and n:
            own_place = torch.arange(n, device="cuda") + (length - n)
            place = torch.arange(length, device="cuda")
            seen = torch.ones(n, length, dtype=torch.bool, device="cuda")
            if c["kind"] != "attend" or c["causal"]:
                seen &= place[None, :] <= own_place[:, None]
                if c["window"]:
                    seen &= own_place[:, None] - place[None, :] < c["window"]
            for h in range(c["heads"]):
                a = x[:, h] @ k[:, h // group].t().contiguous() * (c["dim"] ** -0.5)
                a = torch.softmax(a.masked_fill(~seen, -1e300), dim=1).masked_fill(~seen, 0.0)
                y[:, h] = a @ v[:, h // group].contiguous()
        out.append(y)
    return torch.cat(out)


def _too_long(c):
    return work(c)["flops"] > 4e11 or sum(_sizes(c)[0]) * c["kv"] * c["dim"] > 3e9 or c["entries"] * c["heads"] > 16384


def _exact_decode(c, seed):
    return None if _too_long(c) else {"out": _exact_rows(c, seed, False)}


def _exact_step(c, seed):
    if _too_long(c):
        return None
    _, k, v = _rows(c, c["entries"], seed)
    return {"out": _exact_rows(c, seed, True), "k": _q4_0(k), "v": _q4_0(v)}


def _exact_attend(c, seed):
    return None if _too_long(c) else {"out": _exact_rows(c, seed, False)}
