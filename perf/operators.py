"""A cache in pages held in 4 bits, the attention over it, its pages' bookkeeping, and sampling: the calls of a server that keeps
several sequences, as timed and compared cases.

Four kinds:

  write   new keys, values and queries of several sequences: rotated, the keys and values stored in 4 bits and read back
  attend  queries of the sequences' last tokens over the cache: single tokens, a few, or prompts
  pages   the bookkeeping between steps: sequences forked, grown and freed, or the pool compacted
  sample  the next token of each sequence from its logits and a given random number

A page holds `page` tokens of every layer and KV head, in units of 16 tokens of one head (UNIT below says where a unit keeps what).
An element stands for the fp16 number nearest to d q + m, with one pair of fp16 numbers (d, m) per token and 32 elements.
Random numbers are inputs, sequences have lengths of their own, and pages are scattered over the pool as a running server leaves them.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

NO_PAGE = -1
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
SHIFTS = (0, 16, 4, 20, 8, 24, 12, 28)  # where a word of keys keeps its eight elements


def listed():
    heads = {"heads": 32, "kv_heads": 8, "head": 128, "page": 64}  # the head layout of this package's default decoder
    return [
        # one step of 64 sequences decoded together: a few hundred KB, so the launches count
        {"name": "write_step_64", "kind": "write", **heads, "type": "f32", "seqs": 64, "new": 1, "longest": 2048, "pairing": 0, "rot": 128},
        # the prompts of eight new sequences, lengths as they come, neighbours rotated as some models do, over part of a head
        {"name": "write_prompts", "kind": "write", **heads, "type": "bf16", "seqs": 8, "new": 2048, "longest": 2300, "pairing": 1, "rot": 64},
        # one sequence in the middle of the default decoder's cache: the latency of a single reply
        {"name": "attend_one", "kind": "attend", **heads, "type": "f32", "seqs": 1, "new": 1, "longest": 1500, "window": 0},
        # a busy server's step: 64 sequences of up to 8192 tokens
        {"name": "attend_step_64", "kind": "attend", **heads, "type": "bf16", "seqs": 64, "new": 1, "longest": 8192, "window": 0},
        # two very long sequences: little work but along their tokens
        {"name": "attend_long", "kind": "attend", **heads, "type": "f16", "seqs": 2, "new": 1, "longest": 131072, "window": 0},
        # a 512-token prompt in 32 bits, as the default decoder feeds it
        {"name": "attend_prompt_512", "kind": "attend", **heads, "type": "f32", "seqs": 1, "new": 512, "longest": 512, "window": 0},
        # ragged prompts behind what their sequences hold already
        {"name": "attend_prompts", "kind": "attend", **heads, "type": "bf16", "seqs": 4, "new": 2048, "longest": 4096, "window": 0},
        # four sequences forked to two continuations each, grown by a token and freed: the smallest bookkeeping
        {"name": "pages_fork", "kind": "pages", "what": "fork", "pages": 256, "page_bytes": 81920, "page": 16, "seqs": 4, "ways": 2, "longest": 500},
        # a pool of 1.3 GB, half empty after many sequences have ended, moved together
        {"name": "pages_compact", "kind": "pages", "what": "compact", "pages": 4096, "page_bytes": 327680, "page": 64, "seqs": 48, "ways": 1, "longest": 3500},
        # one reply's token from the default decoder's vocabulary
        {"name": "sample_one", "kind": "sample", "type": "f32", "rows": 1, "vocab": 32000, "filter": "all"},
        # a step of 64 sequences, each with its own settings
        {"name": "sample_64", "kind": "sample", "type": "f32", "rows": 64, "vocab": 32000, "filter": "mixed"},
        # a large batch over a large vocabulary without cut-offs: every logit has a part in the choice
        {"name": "sample_256_wide", "kind": "sample", "type": "bf16", "rows": 256, "vocab": 128256, "filter": "none"},
    ]


def _log_int(rng, lo, hi, step=1):
    """A multiple of `step` between lo and hi, spread over the logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step) * step))


def draw(rng):
    kind = rng.choice(["write", "attend", "attend", "attend", "pages", "sample", "sample"])
    kv = rng.choice([1, 2, 4, 5, 8, 16])
    heads = {"heads": kv * rng.choice([1, 2, 3, 4, 7, 8]), "kv_heads": kv, "head": rng.choice([40, 64, 80, 96, 128, 128, 128, 192, 256]),
             "page": rng.choice([16, 32, 64, 128])}
    if kind == "write":
        new = rng.choice([1, 1, 4, _log_int(rng, 16, 1500)])
        seqs = _log_int(rng, 1, 128 if new < 16 else max(1, 8192 // new))
        rot = rng.choice([heads["head"], heads["head"] // 2, 0])
        return {"kind": kind, **heads, "type": rng.choice(["f32", "f16", "bf16"]), "seqs": seqs, "new": new, "longest": new + _log_int(rng, 1, 2000),
                "pairing": rng.choice([0, 1]), "rot": rot}
    if kind == "attend":
        new = rng.choice([1, 1, 1, rng.randint(2, 8), _log_int(rng, 16, 1500)])
        most = 2_000_000 if new < 16 else 4096  # tokens of all sequences together, times KV heads and elements over 1024
        size = max(1.0, heads["kv_heads"] * heads["head"] / 1024)
        longest = new + _log_int(rng, 16, min(100_000, int(most / size / 8)))
        per = longest if new < 16 else new * max(1.0, longest / 2048) * max(1.0, heads["heads"] / 32)
        seqs = _log_int(rng, 1, max(1, min(128, int((400_000 if new < 16 else 6000) / size / per))))
        return {"kind": kind, **heads, "type": rng.choice(["f32", "f16", "bf16"]), "seqs": seqs, "new": new, "longest": longest,
                "window": rng.choice([0, 0, _log_int(rng, 16, longest)])}
    if kind == "pages":
        what, page, pages = rng.choice(["fork", "fork", "compact"]), rng.choice([16, 32, 64, 128]), _log_int(rng, 64, 4096)
        ways = rng.randint(1, 8) if what == "fork" else 1
        seqs = rng.randint(1, max(1, min(64, pages // (4 * (1 + ways))))) if what == "fork" else rng.randint(2, min(48, pages // 8))
        return {"kind": kind, "what": what, "pages": pages, "page_bytes": _log_int(rng, 16, 327680, 16), "page": page, "seqs": seqs, "ways": ways,
                "longest": max(2, pages * page // (2 * seqs))}
    rows = _log_int(rng, 1, 256)
    return {"kind": kind, "type": rng.choice(["f32", "f16", "bf16"]), "rows": rows, "vocab": _log_int(rng, 1000, min(200_000, 32_000_000 // rows)),
            "filter": rng.choice(["none", "all", "mixed", "mixed"])}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _padded(head):
    return (head + 63) // 64 * 64


def _lengths(c):
    """(length, new tokens) of each sequence: the first the longest, the others spread below it, the same ones for every seed."""
    r = np.random.default_rng(c["longest"] * 1009 + c["seqs"])
    length = np.maximum(1, (c["longest"] * (1 - 0.75 * r.random(c["seqs"]))).astype(np.int64))
    new = np.maximum(1, (c["new"] * (1 - 0.5 * r.random(c["seqs"]))).astype(np.int64))
    length[0], new[0] = c["longest"], c["new"]
    return np.maximum(length, new), new


def _tables(length, page, r, spare=3):
    """Pages of the sequences in a random order over a pool that holds `spare` more."""
    need = (length + page - 1) // page
    n = int(need.sum()) + spare
    order = r.permutation(n).astype(np.int32)
    tables = np.full((len(length), int(need.max()) + 1), NO_PAGE, dtype=np.int32)
    at = 0
    for s, k in enumerate(need):
        tables[s, :k] = order[at: at + k]
        at += k
    return tables, n


def _pool(n, kv_heads, page, dp, g):
    """Pages of a cache as a running model leaves them: random nibbles, scales of values with a spread of about one, and keys with
    a few elements that are larger in every token."""
    units = n * kv_heads * page // 16
    pool = torch.randint(0, 256, (units, 20 * dp), dtype=torch.uint8, device="cuda", generator=g)
    groups = dp // 32
    big = 1 + 3 * (torch.rand(groups, device="cuda", generator=g) < 0.2).float()
    d = (0.18 + 0.12 * torch.rand(units, 16, groups, device="cuda", generator=g)) * big
    m = -d * (7.5 + 1.5 * torch.randn(units, 16, groups, device="cuda", generator=g))
    pool[:, 16 * dp: 18 * dp] = torch.stack([d, m], -1).half().reshape(units, -1).view(torch.uint8)
    d = 0.18 + 0.12 * torch.rand(units, groups, 4, 4, device="cuda", generator=g)
    m = -d * (7.5 + 1.5 * torch.randn(units, groups, 4, 4, device="cuda", generator=g))
    pool[:, 18 * dp: 20 * dp] = torch.stack([d, m], -2).half().reshape(units, -1).view(torch.uint8)
    return pool.view(n, kv_heads * (page // 16) * 20 * dp)


def prepare(case, seed):
    c, r = case, np.random.default_rng(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    cuda = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    st = {"case": c, "status": torch.zeros(1, dtype=torch.int32, device="cuda")}
    if c["kind"] in ("write", "attend"):
        dp, t = _padded(c["head"]), TYPES[c["type"]]
        length, new = _lengths(c)
        if c["new"] == 1:
            new[:] = 1
        tables, n = _tables(length, c["page"], r)
        rows = int(new.sum())
        starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        st.update(pool=_pool(n, c["kv_heads"], c["page"], dp, g), tables=cuda(tables), lengths=cuda(length.astype(np.int32)), starts=cuda(starts),
                  refs=torch.zeros(n, dtype=torch.int32, device="cuda"), rows=rows)
        if c["kind"] == "write":
            # rows of one stacked projection: queries, keys with a few larger elements, values
            width = (c["heads"] + 2 * c["kv_heads"]) * c["head"]
            qkv = torch.randn(rows, width, device="cuda", generator=g)
            qkv *= 1 + 4 * (torch.rand(width, device="cuda", generator=g) < 0.03).float()
            st["qkv"] = qkv.to(t)
            if c["rot"]:
                f = 10000.0 ** (-np.arange(c["rot"] // 2) * 2 / c["rot"])
                a = np.arange(int(length.max()) + 8)[:, None] * f[None, :]
                st["cos"], st["sin"] = cuda(np.cos(a).astype(np.float32)), cuda(np.sin(a).astype(np.float32))
            else:
                st["cos"] = st["sin"] = None
        else:
            # queries that prefer some keys clearly, as trained ones do
            st["q"] = (1.5 * torch.randn(rows, c["heads"] * c["head"], device="cuda", generator=g)).to(t)
        return st
    if c["kind"] == "pages":
        slots, page = c["seqs"] * (1 + c["ways"]), c["page"]
        st["pool"] = torch.randint(0, 256, (c["pages"], c["page_bytes"]), dtype=torch.uint8, device="cuda", generator=g)
        length, _ = _lengths({**c, "new": 1})
        while (-(-length // page)).sum() > c["pages"] - 2 * slots and length.max() > 1:  # room for what the sequences grow by
            length = np.maximum(1, length // 2)
        need = -(-length // page)
        order = r.permutation(c["pages"]).astype(np.int32)
        tables = np.full((slots, int(need.max()) + 4), NO_PAGE, dtype=np.int32)
        lengths, refs = np.zeros(slots, dtype=np.int32), np.zeros(c["pages"], dtype=np.int32)
        at = 0
        for s in range(c["seqs"]):
            tables[s, : need[s]] = order[at: at + need[s]]
            lengths[s] = length[s]
            at += need[s]
        refs[order[:at]] = 1
        st.update(tables0=cuda(tables), lengths0=cuda(lengths), refs0=cuda(refs))
        st.update(tables=st["tables0"].clone(), lengths=st["lengths0"].clone(), refs=st["refs0"].clone())
        src = np.repeat(np.arange(c["seqs"]), c["ways"]).astype(np.int32)
        dst = (c["seqs"] + np.arange(c["seqs"] * c["ways"])).astype(np.int32)
        every = np.arange(slots).astype(np.int32)
        grow = r.integers(1, 3, slots).astype(np.int32)
        gone = np.arange(0, c["seqs"], 2).astype(np.int32)
        st.update(src=cuda(src), dst=cuda(dst), every=cuda(every), grow=cuda(grow), gone=cuda(gone))
        return st
    rows, vocab = c["rows"], c["vocab"]
    # logits of a spread of 2.5 with a few clear favourites a row
    x = 2.5 * torch.randn(rows, vocab, device="cuda", generator=g)
    x.scatter_add_(1, torch.randint(0, vocab, (rows, 20), device="cuda", generator=g), 4 + 3 * torch.randn(rows, 20, device="cuda", generator=g))
    st["logits"] = x.to(TYPES[c["type"]])
    st["u"] = torch.rand(rows, device="cuda", generator=g)
    pick = lambda *a: cuda(r.choice(a, rows).astype(np.float32))  # noqa: E731
    if c["filter"] == "none":
        st.update(temperature=pick(0.7, 1.0, 1.3), top_k=None, top_p=None, min_p=None)
    elif c["filter"] == "all":
        st.update(temperature=pick(0.8), top_k=pick(50).int(), top_p=pick(0.95), min_p=pick(0.02))
    else:
        st.update(temperature=pick(0.0, 0.6, 0.8, 1.0, 1.5), top_k=pick(0, 0, 1, 20, 50, 1000).int(), top_p=pick(1.0, 0.9, 0.95, 0.5),
                  min_p=pick(0.0, 0.0, 0.05, 0.1))
    return st


# ---- the plain forms -------------------------------------------------------------------------------------------------
def _unit_places(dp):
    """UNIT: where the 16 tokens of one head are within 20 dp bytes.  Keys: byte and bit of element i of token t; values: the same;
    then, counted in fp16 numbers, the (d, m) of token t and group g of the keys and of the values."""
    t, i, groups = np.arange(16)[:, None], np.arange(dp)[None, :], dp // 32
    w = 4 if dp % 128 == 0 else 2  # words of one quarter that lie together
    j, quarter, e = i // 32, i % 32 // 8, i % 8
    bit = np.array(SHIFTS)[e]
    kb = t * (dp // 2) + 4 * (j // w * 4 * w + quarter * w + j % w) + bit // 8
    tile, dim = i // 16, i % 16
    vb = 8 * dp + 4 * (tile // 4 * 128 + (dim % 8 * 4 + t // 4) * 4 + tile % 4) + np.array([0, 2, 1, 3])[t % 4]
    vs = dim // 8 * 4 + 0 * t
    g = np.arange(groups)[None, :]
    kd = 8 * dp + 2 * (t * groups + g)
    vd = 9 * dp + 8 * (g * 4 + t // 4) + t % 4
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(np.broadcast_to(a, np.broadcast_shapes(a.shape, (16, 1))))).long().cuda()  # noqa: E731
    return {"k": (dev(kb), dev(bit % 8 + 0 * t)), "v": (dev(vb), dev(vs)), "kd": dev(kd), "km": dev(kd + 1), "vd": dev(vd), "vm": dev(vd + 4)}


def _values(units, dp, which, places):
    """Values [..., 16, dp] in fp32 of units [..., 20 dp] bytes."""
    b, s = places[which]
    q = (units[..., b.view(-1)].view(*units.shape[:-1], 16, dp) >> s.to(torch.uint8)) & 15
    halves = units.view(torch.float16)
    d, m = (halves[..., places[which + x].view(-1)].view(*units.shape[:-1], 16, dp // 32).float() for x in "dm")
    return (q.float().view(*q.shape[:-1], dp // 32, 32) * d[..., None] + m[..., None]).half().float().flatten(-2)


def _cache_rows(st, which, places):
    """[sequences, kv heads, tokens, head] of all pages in the tables; what is past a sequence's pages is of no meaning."""
    c = st["case"]
    dp, page = _padded(c["head"]), c["page"]
    pages = st["pool"][st["tables"].clamp(min=0).long()].view(*st["tables"].shape, c["kv_heads"], page // 16, 20 * dp)
    return _values(pages, dp, which, places).permute(0, 2, 1, 3, 4, 5).flatten(2, 4)[..., : c["head"]]


def _row_places(st):
    """For every new row: its sequence and its position."""
    rows = torch.arange(st["rows"], device="cuda")
    seq = torch.searchsorted(st["starts"][1:].long(), rows, right=True)
    new = (st["starts"][1:] - st["starts"][:-1]).long()
    return seq, st["lengths"].long()[seq] - new[seq] + rows - st["starts"].long()[seq]


def _rotated(x, pos, st):
    """x [rows, heads, head] in fp32."""
    c = st["case"]
    if not c["rot"]:
        return x
    cos, sin = st["cos"][pos][:, None], st["sin"][pos][:, None]
    r, y = c["rot"], x.clone()
    a, b = (slice(0, r, 2), slice(1, r, 2)) if c["pairing"] else (slice(0, r // 2), slice(r // 2, r))
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., a] * sin + x[..., b] * cos
    return y


def _codes(x, dp):
    """x [rows, heads, head] -> codes [rows, heads, dp], d and m [rows, heads, groups]; the last group may be short."""
    x = torch.nan_to_num(x, nan=0.0, posinf=32768.0, neginf=-32768.0).clamp(-32768, 32768)
    pad = dp - x.shape[-1]
    lo = torch.nn.functional.pad(x, (0, pad), value=math.inf).unflatten(-1, (-1, 32)).amin(-1)
    hi = torch.nn.functional.pad(x, (0, pad), value=-math.inf).unflatten(-1, (-1, 32)).amax(-1)
    lo, hi = torch.where(lo == math.inf, 0.0, lo), torch.where(hi == -math.inf, 0.0, hi)
    m = lo.half()
    d = ((hi - m.float()) / torch.full((), 15.0, device="cuda")).half()  # (a Python number would be multiplied by its reciprocal)
    d = torch.where(d > 0, d, 0.0).half()
    v = (torch.nn.functional.pad(x, (0, pad)).unflatten(-1, (-1, 32)) - m.float()[..., None]) / d.float()[..., None]
    q = torch.where(d[..., None] > 0, torch.round(v).clamp(0, 15), 0.0).flatten(-2)
    return torch.where(torch.arange(dp, device="cuda") < x.shape[-1], q, 0.0).to(torch.uint8), d, m


def _plain_write(st):
    c = st["case"]
    dp, page, nh, kv, hd = _padded(c["head"]), c["page"], c["heads"], c["kv_heads"], c["head"]
    places = _unit_places(dp)
    seq, pos = _row_places(st)
    x = st["qkv"].float()
    q = _rotated(x[:, : nh * hd].view(-1, nh, hd), pos, st)
    k = _rotated(x[:, nh * hd: (nh + kv) * hd].view(-1, kv, hd), pos, st)
    v = x[:, (nh + kv) * hd:].view(-1, kv, hd)
    pageno = st["tables"][seq, pos // page].long()
    unit = ((pageno[:, None] * kv + torch.arange(kv, device="cuda")) * (page // 16) + (pos % page // 16)[:, None]) * 20 * dp  # [rows, kv]
    row, flat, halves = pos % 16, st["pool"].view(-1), st["pool"].view(-1).view(torch.float16)
    out = []
    for which, y, step in (("k", k, 2), ("v", v, 8)):
        code, d, m = _codes(y, dp)
        low = torch.arange(dp, device="cuda")
        low = low[low // step % 2 == 0]  # a byte keeps elements i and i + step
        flat[unit[..., None] + places[which][0][row][:, None, low]] = code[..., low] | code[..., low + step] << 4
        halves[unit[..., None] // 2 + places[which + "d"][row][:, None]] = d
        halves[unit[..., None] // 2 + places[which + "m"][row][:, None]] = m
    for which in "kv":
        units = flat[unit[..., None] + torch.arange(20 * dp, device="cuda")]
        vals = _values(units, dp, which, places)  # [rows, kv, 16, dp]
        vals = vals[torch.arange(st["rows"], device="cuda"), :, row]
        out.append(vals[..., :hd].half().flatten(1))
    return {"q": q.flatten(1).to(st["qkv"].dtype), "k": out[0], "v": out[1]}


def _plain_attend(st):
    c = st["case"]
    nh, kv, hd, rep = c["heads"], c["kv_heads"], c["head"], c["heads"] // c["kv_heads"]
    places = _unit_places(_padded(hd))
    seq, pos = _row_places(st)
    at = torch.arange(st["rows"], device="cuda") - st["starts"].long()[seq]
    width, n = c["new"], st["lengths"].shape[0]
    q = torch.zeros(n, width, nh, hd, device="cuda")
    q[seq, at] = st["q"].float().view(-1, nh, hd)
    where = torch.full((n, width), -1, dtype=torch.long, device="cuda")
    where[seq, at] = pos
    q = q.view(n, width, kv, rep, hd).permute(0, 2, 3, 1, 4).reshape(n, kv, rep * width, hd)
    k = _cache_rows(st, "k", places)
    keys = torch.arange(k.shape[2], device="cuda")
    s = q @ k.transpose(-1, -2) * float(np.float32(hd ** -0.5))
    del k
    sees = keys <= where[..., None]
    if c["window"]:
        sees &= where[..., None] - keys < c["window"]
    s = s.view(n, kv, rep, width, -1).masked_fill_(~sees[:, None, None], -math.inf).view(n, kv, rep * width, -1)
    top = s.amax(-1, keepdim=True)
    s = s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = s.sum(-1, keepdim=True)
    v = _cache_rows(st, "v", places)
    v.masked_fill_((keys >= st["lengths"].long()[:, None])[:, None, :, None], 0.0)
    y = s @ v / torch.where(total == 0, 1.0, total)
    y = y.view(n, kv, rep, width, hd).permute(0, 3, 1, 2, 4).reshape(n, width, nh * hd)
    return y[seq, at].to(st["q"].dtype)


def _plain_pages(st):
    c = st["case"]
    page, n_pages = c["page"], c["pages"]
    st["tables"].copy_(st["tables0"])
    st["lengths"].copy_(st["lengths0"])
    st["refs"].copy_(st["refs0"])
    tables, lengths, refs, pool = st["tables"], st["lengths"], st["refs"], st["pool"]
    width = tables.shape[1]
    columns = torch.arange(width, device="cuda")
    count = lambda rows: -(-lengths[rows].long() // page)  # noqa: E731

    def free(rows):
        held = columns < count(rows)[:, None]
        refs.scatter_add_(0, tables[rows].clamp(min=0).long().view(-1), -held.int().view(-1))
        tables[rows], lengths[rows] = NO_PAGE, 0

    if c["what"] == "fork":
        src, dst = st["src"].long(), st["dst"].long()
        held = columns < count(src)[:, None]
        tables[dst] = torch.where(held, tables[src], NO_PAGE)
        lengths[dst] = lengths[src]
        refs.scatter_add_(0, tables[src].clamp(min=0).long().view(-1), held.int().view(-1))
        rows, grow = st["every"].long(), st["grow"].long()
        have, want = count(rows), -(-(lengths[rows].long() + grow) // page)
        last = tables[rows, (have - 1).clamp(min=0)].clamp(min=0).long()
        partial = lengths[rows] % page != 0
        # of the growing sequences that share a page, all but the last holder copy it
        earlier = ((last[None, :] == last[:, None]) & partial[None, :] & partial[:, None]).tril(-1).sum(-1)
        copied = partial & (refs[last] - earlier > 1)
        need = want - have + copied.long()
        first = torch.cumsum(need, 0) - need
        fresh = torch.nonzero(refs == 0).view(-1)
        at = columns - have[:, None] + copied.long()[:, None]  # which of a sequence's new pages goes to a column
        new = (at >= 0) & (columns < want[:, None]) & (need > 0)[:, None]
        index = (first[:, None] + at)[new]
        tables[rows] = torch.where(new, 0, tables[rows])
        tables[rows[:, None].expand(-1, width)[new], columns[None].expand(len(rows), -1)[new]] = fresh[index].int()
        refs[fresh[: int(need.sum())]] = 1
        refs.scatter_add_(0, last, -copied.int())
        pool[fresh[first[copied]]] = pool[last[copied]]
        lengths[rows] += grow.int()
        free(st["gone"].long())
    else:
        free(st["gone"].long())
        live = torch.nonzero(refs > 0).view(-1)
        n = len(live)
        holes = torch.nonzero(refs[:n] == 0).view(-1)
        late = live[live >= n]
        to = torch.arange(n_pages, device="cuda", dtype=torch.int32)
        to[late] = holes.int()
        pool[holes] = pool[late]
        refs[holes], refs[late] = refs[late], 0
        tables.copy_(torch.where(tables >= 0, to[tables.clamp(min=0).long()], tables))
    return {"tables": tables, "lengths": lengths, "refs": refs, "pool": pool}


def _plain_sample(st):
    x = st["logits"].double()
    rows, vocab = x.shape
    column = lambda name, fill: st[name].double()[:, None] if st[name] is not None else torch.full((rows, 1), fill, dtype=torch.float64, device="cuda")  # noqa: E731
    t, k, p, least = column("temperature", 1.0), column("top_k", 0), column("top_p", 1.0), column("min_p", 0.0)
    greedy = t == 0
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    w = torch.exp((x - x.amax(1, keepdim=True)) / torch.where(greedy, 1.0, t))
    sorted_w = w.gather(1, order)
    rank = torch.arange(vocab, device="cuda")
    kept = (rank < torch.where((k <= 0) | greedy, torch.where(greedy, 1.0, float(vocab)), k))
    sorted_w = torch.where(kept, sorted_w, 0.0)
    before = torch.cumsum(sorted_w, 1) - sorted_w
    kept &= (before < p * sorted_w.sum(1, keepdim=True)) | (p >= 1) | (rank == 0)
    kept &= (sorted_w >= least) | (rank == 0)
    keep = torch.zeros_like(kept).scatter_(1, order, kept)
    w = torch.where(keep, w, 0.0)
    sums = torch.cumsum(w, 1)
    total = sums[:, -1:]
    token = (sums > st["u"].double()[:, None] * total).int().argmax(1)
    return {"tokens": token.int(), "logprobs": torch.log(w.gather(1, token[:, None]) / total).view(-1).float()}


# ---- the framework's calls -------------------------------------------------------------------------------------------
def _own(st):
    from cut_b200 import ops
    from cut_b200.paged import PagedCache

    c, status = st["case"], st["status"]
    if c["kind"] == "sample":
        tokens, logprobs = ops.sample(st["logits"], st["u"], temperature=st["temperature"], top_k=st["top_k"], top_p=st["top_p"], min_p=st["min_p"],
                                      want_logprobs=True, status=status)
        return {"tokens": tokens, "logprobs": logprobs}
    if c["kind"] == "pages":
        cache = PagedCache(st["pool"], st["tables"], st["lengths"], st["refs"], page_tokens=c["page"], status=status)
        cache.tables.copy_(st["tables0"])
        cache.lengths.copy_(st["lengths0"])
        cache.refs.copy_(st["refs0"])
        if c["what"] == "fork":
            cache.fork(st["src"], st["dst"])
            cache.reserve(st["every"], st["grow"])
            cache.free(st["gone"])
        else:
            cache.free(st["gone"])
            cache.compact()
        return {"tables": cache.tables, "lengths": cache.lengths, "refs": cache.refs, "pool": cache.pages}
    cache = PagedCache(st["pool"], st["tables"], st["lengths"], st["refs"], page_tokens=c["page"], n_kv_heads=c["kv_heads"], head_dim=c["head"], status=status)
    starts = None if c["new"] == 1 else st["starts"]
    if c["kind"] == "attend":
        return ops.paged_attention(cache, st["q"], c["heads"], starts=starts, max_new=c["new"], window=c["window"])
    a, b = c["heads"] * c["head"], (c["heads"] + c["kv_heads"]) * c["head"]
    q, k, v = st["qkv"][:, :a], st["qkv"][:, a:b], st["qkv"][:, b:]
    q = ops.paged_kv_write(cache, k, v, starts=starts, q=q, cos_t=st["cos"], sin_t=st["sin"], rot_dims=c["rot"], pairing=c["pairing"])
    k, v = ops.paged_kv_read(cache, st["rows"], starts=starts, dtype=torch.float16)
    return {"q": q, "k": k, "v": v}


def run(state):
    if own:
        return _own(state)
    return {"write": _plain_write, "attend": _plain_attend, "pages": _plain_pages, "sample": _plain_sample}[state["case"]["kind"]](state)


# ---- what a pass cannot do without -------------------------------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] == "sample":
        return {"bytes": c["rows"] * (c["vocab"] * BYTES[c["type"]] + 28), "flops": c["rows"] * c["vocab"]}
    if c["kind"] == "pages":
        mean = 0.625 * c["longest"] * c["seqs"]
        live = 0.5 * mean / c["page"]
        moved = c["seqs"] * c["ways"] if c["what"] == "fork" else live * (1 - live / c["pages"])
        return {"bytes": int(2 * moved * c["page_bytes"] + 4 * c["pages"] + 8 * mean / c["page"]), "flops": 0}
    rows = c["seqs"] * (1 if c["new"] == 1 else 0.75 * c["new"])
    token = 1.25 * c["kv_heads"] * c["head"]  # bytes of a token's keys and values in the cache
    if c["kind"] == "write":
        width = (c["heads"] + 2 * c["kv_heads"]) * c["head"]
        read = 4 * c["kv_heads"] * c["head"]
        return {"bytes": int(rows * (width * BYTES[c["type"]] + c["heads"] * c["head"] * BYTES[c["type"]] + token + read + 4 * c["rot"])), "flops": int(rows * width * 6)}
    length = max(c["new"], 0.625 * c["longest"] if c["seqs"] > 1 else c["longest"])
    seen = length - (rows / c["seqs"] - 1) / 2  # keys of a query
    if c["window"]:
        seen = min(seen, c["window"])
    read = min(length, seen + rows / c["seqs"])
    return {"bytes": int(c["seqs"] * read * token + 2 * rows * c["heads"] * c["head"] * BYTES[c["type"]]),
            "flops": int(4 * rows * c["heads"] * c["head"] * seen)}


# ---- the definitions in 64 bits, apart from the above ------------------------------------------------------------------
def _f32(x):
    return x.float().double()


def _to_half(x):
    """The fp16 number nearest to a float64 one, in float64 (ties to even)."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -14)))
    e = torch.where(x.abs() >= torch.exp2(e + 1), e + 1, e)
    step = torch.exp2(e - 10)
    return torch.round(x / step) * step


def _exact_head(units, dp, which):
    """Units [n, 20 dp] bytes of one head -> float64 [16 n, dp], element by element from the layout's description."""
    n, groups = units.shape[0], dp // 32
    out = torch.empty(n, 16, dp, dtype=torch.float64, device="cuda")
    halves = units.view(torch.float16).double()
    for g in range(groups):
        for b in range(4):  # eight elements of the group at a time
            for e in range(8):
                i = 32 * g + 8 * b + e
                for t in range(16):
                    if which == "k":
                        w = 4 if dp % 128 == 0 else 2
                        word = t * (dp // 8) + g // w * 4 * w + b * w + g % w
                        q = units[:, 4 * word + SHIFTS[e] // 8].long() >> (SHIFTS[e] % 8) & 15
                        d, m = halves[:, 8 * dp + 2 * (t * groups + g)], halves[:, 8 * dp + 2 * (t * groups + g) + 1]
                    else:
                        word = 2 * dp + i // 64 * 128 + (i % 8 * 4 + t // 4) * 4 + i // 16 % 4
                        q = units[:, 4 * word + (0, 2, 1, 3)[t % 4]].long() >> (4 * (i // 8 % 2)) & 15
                        d, m = halves[:, 9 * dp + 8 * (g * 4 + t // 4) + t % 4], halves[:, 9 * dp + 8 * (g * 4 + t // 4) + 4 + t % 4]
                    out[:, t, i] = d * q + m
    return _to_half(out).view(n * 16, dp)


def _exact_attend(st):
    c = st["case"]
    dp, page, hd, kv, rep = _padded(c["head"]), c["page"], c["head"], c["kv_heads"], c["heads"] // c["kv_heads"]
    starts, lengths = st["starts"].tolist(), st["lengths"].tolist()
    y = torch.zeros(st["rows"], c["heads"], hd, dtype=torch.float64, device="cuda")
    q = st["q"].double().view(-1, c["heads"], hd)
    scale = float(np.float32(hd ** -0.5))
    pool = st["pool"].view(-1, kv, page // 16, 20 * dp)
    pages = [st["tables"][s, : -(-lengths[s] // page)].long() for s in range(c["seqs"])]
    cut = np.cumsum([0] + [len(p) * page for p in pages])
    for h in range(kv):
        units = pool[torch.cat(pages), h].reshape(-1, 20 * dp)
        keys, values = _exact_head(units, dp, "k"), _exact_head(units, dp, "v")
        for s in range(c["seqs"]):
            a, b, n = starts[s], starts[s + 1], lengths[s]
            k, v = keys[cut[s]: cut[s] + n, :hd], values[cut[s]: cut[s] + n, :hd]
            at = torch.arange(n - (b - a), n, device="cuda")[:, None]
            j = torch.arange(n, device="cuda")[None, :]
            sees = j <= at
            if c["window"]:
                sees = sees & (at - j < c["window"])
            for r in range(rep):
                p = torch.softmax((q[a:b, h * rep + r] @ k.T * scale).masked_fill(~sees, -math.inf), -1)
                y[a:b, h * rep + r] = p @ v
    return y.flatten(1)


def _exact_write(st):
    c = st["case"]
    nh, kv, hd = c["heads"], c["kv_heads"], c["head"]
    starts, lengths = st["starts"].cpu().numpy(), st["lengths"].cpu().numpy()
    pos = np.concatenate([np.arange(lengths[s] - (starts[s + 1] - starts[s]), lengths[s]) for s in range(c["seqs"])])
    x = st["qkv"].double().view(-1, nh + 2 * kv, hd)
    if c["rot"]:
        p = torch.from_numpy(pos).cuda()
        for i in range(c["rot"] // 2):
            a, b = (2 * i, 2 * i + 1) if c["pairing"] else (i, i + c["rot"] // 2)
            cs, sn = st["cos"][p, i].double()[:, None], st["sin"][p, i].double()[:, None]
            u, w = x[:, : nh + kv, a].clone(), x[:, : nh + kv, b].clone()
            x[:, : nh + kv, a] = _f32(_f32(u * cs) - _f32(w * sn))  # (products of fp32 numbers are exact in float64: one rounding each)
            x[:, : nh + kv, b] = _f32(_f32(u * sn) + _f32(w * cs))
    y = x[:, nh:].clamp(-32768, 32768)
    out = torch.empty_like(y)
    for g in range(0, hd, 32):
        part = y[..., g: g + 32]
        m = _to_half(part.amin(-1, keepdim=True))
        d = _to_half(_f32(_f32(part.amax(-1, keepdim=True) - m) / 15)).clamp(min=0)
        q = torch.where(d > 0, torch.round(_f32(_f32(part - m) / torch.where(d > 0, d, 1.0))).clamp(0, 15), 0.0)
        out[..., g: g + 32] = _to_half(d * q + m)
    return {"q": x[:, :nh].flatten(1), "k": out[:, :kv].flatten(1), "v": out[:, kv:].flatten(1)}


def _exact_sample(st):
    x = st["logits"].double().cpu().numpy()
    get = lambda name, fill: st[name].double().cpu().numpy() if st[name] is not None else np.full(len(x), fill)  # noqa: E731
    t, k, p, least, u = get("temperature", 1.0), get("top_k", 0), get("top_p", 1.0), get("min_p", 0.0), st["u"].double().cpu().numpy()
    tokens, logprobs = np.zeros(len(x), dtype=np.int32), np.zeros(len(x))
    for r, row in enumerate(x):
        if t[r] == 0:
            tokens[r] = int(np.argmax(row))
            continue
        order = np.argsort(-row, kind="stable")
        w = np.exp((row[order] - row[order[0]]) / t[r])
        if 0 < k[r] < len(row):
            order, w = order[: int(k[r])], w[: int(k[r])]
        if p[r] < 1:
            n = max(1, int(np.searchsorted(np.cumsum(w), p[r] * math.fsum(w), side="left")) + 1)
            order, w = order[:n], w[:n]
        n = max(1, int(np.count_nonzero(w >= least[r])))
        order, w = order[:n], w[:n]
        by_index = np.argsort(order)
        sums = np.cumsum(w[by_index])
        i = min(int(np.searchsorted(sums, u[r] * sums[-1], side="right")), len(sums) - 1)
        tokens[r], logprobs[r] = order[by_index[i]], math.log(w[by_index[i]] / sums[-1])
    return {"tokens": torch.from_numpy(tokens), "logprobs": torch.from_numpy(logprobs)}


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "attend":
        if case["heads"] * case["head"] * case["seqs"] * case["longest"] * case["new"] > 4e11:
            return None
        return _exact_attend(st)
    if case["kind"] == "write":
        return _exact_write(st)
    return _exact_sample(st) if case["kind"] == "sample" else None
