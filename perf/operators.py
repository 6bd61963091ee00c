"""Timed cases of the paged key-value cache: attention layers that serve many sequences at once.

A case is a dict of plain values; `op` names the operator it goes through:

  rope    coli_hip_qk_rope_paged: norms of query and key heads, rotary positions, and the new
          keys and values written into the pages of their sequences
  attn    coli_hip_attn_paged: one query row per token over the pages of its sequence
  fork    coli_hip_pages_free and coli_hip_pages_fork: the branches of the step before are
          dropped and new ones taken from their parents (shared full pages, or whole copies)
  churn   coli_hip_pages_free, _compact, _append: half of the sequences end, the pool is
          closed up, as many new ones start

The pool is [n_pages][n_layers][2][KH][page][hd]; table[s][j] is the page of positions
j * page .. of sequence s (-1: none), lens[s] its length, refs[p] how many table entries hold
page p.  Page ids are scattered, as after hours of serving; slots past a sequence's end hold
whatever was there (NaN among it).  Sizes are those of the benchmark's attention layers (16
query and 2 key-value heads of 256, 64 rotary columns, gated) and generic ones.
"""
import importlib.util
import math
import os
import random

import torch

own = False

F64 = torch.float64
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2}
EPS = 1e-6


def listed():
    big = {"H": 16, "KH": 2, "hd": 256, "rot": 64, "style": "half", "dtype": "bf16", "page": 16, "layers": 1, "gated": True}
    wide = {"H": 32, "KH": 8, "hd": 128, "rot": 128, "style": "interleaved", "dtype": "f16", "page": 32, "layers": 2,
            "gated": False}
    return [
        # the new token of one request far into a long context: a launch and its latency
        {"name": "rope_1_far", "op": "rope", "n": 1, "per": 1, "len": 131000, "factor": 4.0, **big},
        # a decode step of many requests
        {"name": "rope_192", "op": "rope", "n": 192, "per": 1, "len": 2100, "factor": 1.0, **big},
        # a prefill step: odd chunks of five prompts
        {"name": "rope_4000", "op": "rope", "n": 5, "per": 801, "len": 2500, "factor": 1.0, **wide},
        # one request with a short history: latency
        {"name": "attn_1x600", "op": "attn", "n": 1, "len": 600, "ragged": False, **big},
        # a small batch, full histories
        {"name": "attn_8x4000", "op": "attn", "n": 8, "len": 4000, "ragged": False, **big},
        # an ordinary batch: lengths from nothing to 16000
        {"name": "attn_48_ragged", "op": "attn", "n": 48, "len": 16000, "ragged": True, **big},
        # two requests with whole books: few rows, a long axis
        {"name": "attn_2x120000", "op": "attn", "n": 2, "len": 120000, "ragged": False, **dict(big, dtype="f16")},
        # a large batch of chats, four query heads a key-value head
        {"name": "attn_200_g4", "op": "attn", "n": 200, "len": 2900, "ragged": True, **dict(wide, dtype="bf16")},
        # every head with its own keys, in 32 bits
        {"name": "attn_16_mha_f32", "op": "attn", "n": 16, "len": 3001, "ragged": True, **dict(
            wide, H=8, KH=8, hd=64, rot=64, dtype="f32", page=16)},
        # sampling five continuations of each of twelve prompts
        {"name": "fork_12x5", "op": "fork", "n": 12, "each": 5, "len": 3500, "share": True, **dict(big, layers=10)},
        # six sequences copied whole, before they are edited
        {"name": "copy_6", "op": "fork", "n": 6, "each": 1, "len": 2200, "share": False, **dict(big, layers=10)},
        # half of the requests replaced
        {"name": "churn_40", "op": "churn", "n": 40, "len": 1800, **dict(big, layers=10)},
    ]


HEADS = [(16, 2, 256, 64), (32, 8, 128, 128), (8, 8, 64, 64), (12, 4, 80, 40), (7, 1, 128, 64), (40, 8, 128, 128),
         (10, 10, 112, 112), (20, 1, 176, 64)]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "rope", "attn", "attn", "attn", "attn", "fork", "churn"])
    H, KH, hd, rot = rng.choice(HEADS)
    c = {"op": op, "H": H, "KH": KH, "hd": hd, "rot": rot, "style": rng.choice(["half", "interleaved"]),
         "dtype": rng.choice(["f32", "f16", "bf16", "bf16"]), "page": rng.choice([1, 8, 16, 16, 20, 32, 64, 128]),
         "layers": rng.choice([1, 2, 3]), "gated": rng.random() < 0.5}
    most = 100_000_000 if op == "attn" else 30_000_000   # values of K and V in a layer
    row = 2 * KH * hd
    if op == "rope":
        c.update(n=_log_int(rng, 1, 256), per=rng.choice([1, 1, _log_int(rng, 1, 500)]), factor=rng.choice([1.0, 8.0]))
        c["per"] = max(1, min(c["per"], 4000 // c["n"]))
        c["len"] = c["per"] + _log_int(rng, 1, max(2, min(100_000, most // row // c["n"])))
    elif op == "attn":
        c.update(n=_log_int(rng, 1, 200), ragged=rng.random() < 0.7)
        c["len"] = _log_int(rng, 1, max(2, min(100_000, most // row // c["n"])))
    elif op == "fork":
        c.update(n=_log_int(rng, 1, 32), each=rng.randint(1, 6), share=rng.random() < 0.6)
        c["len"] = _log_int(rng, 1, max(2, min(8000, most // row // (c["n"] * (1 if c["share"] else 1 + c["each"])))))
    else:
        c.update(n=2 * _log_int(rng, 1, 48))
        c["len"] = _log_int(rng, 2, max(3, min(8000, most // row // c["n"])))
    return c


# ---------------------------------------------------------------- what a case's sizes come to
def _lens(case):
    """The length of each sequence: of the case alone, so that its work is known."""
    n, top, rng = case["n"], case["len"], random.Random(case["len"] * 1009 + case["n"])
    if case["op"] == "rope":
        return [top] + [case["per"] + rng.randint(0, top - case["per"]) for _ in range(n - 1)]
    if case["op"] in ("fork", "churn"):
        return [top] + [rng.randint(max(1, top // 2), top) for _ in range(n - 1)]
    if not case["ragged"] or n == 1:
        return [top] * n
    return [top, 0, 1][:min(n, 3)] + [_log_int(rng, max(1, top // 64), top) for _ in range(n - 3)]


def _pages_of(lens, page):
    return [(x + page - 1) // page for x in lens]


def _row_bytes(case):
    """Bytes of one position's K and V in one layer."""
    return 2 * case["KH"] * case["hd"] * (4 if case["dtype"] == "f32" else 2)


def _group(case):
    """The sequences of the half that ends first (0) and of the other (1)."""
    h = case["n"] // 2
    return list(range(h)), list(range(h, 2 * h))


def work(case):
    lens, page, H, hd = _lens(case), case["page"], case["H"], case["hd"]
    pages, row = _pages_of(lens, page), _row_bytes(case)
    if case["op"] == "rope":
        t = case["n"] * case["per"]
        heads = t * (H + case["KH"]) * hd
        return {"bytes": 4 * (2 * t * H * hd + 2 * t * case["KH"] * hd) + t * row + 12 * t, "flops": 8 * heads}
    if case["op"] == "attn":
        n, keys = case["n"], sum(lens)
        return {"bytes": keys * row + 4 * n * H * hd * (3 if case["gated"] else 2) + 4 * sum(pages) + 8 * n,
                "flops": 4 * keys * H * hd}
    if case["op"] == "fork":
        rows = sum((x % page if case["share"] else x) for x in lens) * case["each"]
        return {"bytes": 2 * rows * row * case["layers"] + (8 + 8) * sum(pages) * case["each"], "flops": 0}
    a, b = (sum(pages[s] for s in g) for g in _group(case))
    return {"bytes": 2 * min(a, b) * page * row * case["layers"] + 8 * (a + b), "flops": 0}


# ---------------------------------------------------------------- seeded inputs
def _gen(seed, *tags):
    h = 1469598103934665603
    for v in (seed, *tags):
        h = ((h ^ (int(v) & 0xFFFFFFFF)) * 1099511628211) & 0x7FFFFFFFFFFFFFFF
    return torch.Generator(device="cuda").manual_seed(h)


def _normal(shape, sigma, seed, *tags):
    return torch.randn(shape, device="cuda", generator=_gen(seed, *tags)) * sigma


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _used(refs):
    """The bitmap of pages in use, bit p % 32 of word p // 32."""
    n = refs.numel()
    bits = torch.zeros((n + 31) // 32 * 32, dtype=torch.int64, device="cuda")
    bits[:n] = (refs > 0).long()
    w = (bits.view(-1, 32) << torch.arange(32, device="cuda")).sum(1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).int()


def _pool(case, seed, lens, spare_pages, spare_seqs, spans=None):
    """A pool whose sequences hold `lens` positions; `spans`: groups of sequences whose pages
    lie in regions one after the other (else all are scattered over the pool)."""
    page, dt = case["page"], TYPES[case["dtype"]]
    count = _pages_of(lens, page)
    total = sum(count)
    n_pages, n_seqs, max_pages = total + spare_pages, len(lens) + spare_seqs, max(1, max(count) + 2)
    g = _gen(seed, 1)
    if spans is None:
        ids = torch.randperm(n_pages, device="cuda", generator=g)[:total]
    else:
        parts, at = [], 0
        for s in spans:
            k = sum(count[i] for i in s)
            parts.append(at + torch.randperm(k, device="cuda", generator=g))
            at += k
        ids = torch.cat(parts)
    row = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), torch.tensor(count, device="cuda"))
    first = torch.tensor([sum(count[:i]) for i in range(len(lens))], device="cuda")
    table = torch.full((n_seqs, max_pages), -1, dtype=torch.int32, device="cuda")
    table[row, torch.arange(total, device="cuda") - first[row]] = ids.int()
    refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    refs[ids] = 1
    data = torch.empty((n_pages, case["layers"], 2, case["KH"], page, case["hd"]), dtype=dt, device="cuda")
    step = max(1, (1 << 27) // data[0].numel())
    for a in range(0, n_pages, step):   # keys and values of about unit size, in pieces
        data[a:a + step] = torch.randn(data[a:a + step].shape, device="cuda", generator=g)
    return {"data": data, "table": table, "lens": _ints(lens + [0] * spare_seqs), "refs": refs, "used": _used(refs),
            "state": torch.zeros(16, dtype=torch.int32, device="cuda"),
            "work": torch.empty(n_seqs + 2 * n_pages + 64, dtype=torch.int32, device="cuda")}


def _spoil(case, st, lens):
    """NaN in the slots past each sequence's end."""
    page = case["page"]
    for s, x in enumerate(lens):
        if x % page:
            st["data"][st["table"][s, x // page].long(), :, :, :, x % page:] = float("nan")


def _freq(case):
    """Inverse frequencies [rot / 2]: base 1e7, the slow ones stretched for long contexts."""
    j = torch.arange(case["rot"] // 2, dtype=F64, device="cuda")
    f = 1e7 ** (-2.0 * j / case["rot"])
    if case.get("factor", 1.0) > 1.0:
        mix = (j / (case["rot"] / 2)).clamp(0, 1)
        f = f * (1 - mix) + f / case["factor"] * mix
    return f.float()


def prepare(case, seed):
    lens, H, KH, hd, page = _lens(case), case["H"], case["KH"], case["hd"], case["page"]
    st = {"case": dict(case), "layer": case["layers"] - 1, "turn": 0}
    if case["op"] in ("rope", "attn"):
        st.update(_pool(case, seed, lens, 5, 1))
    if case["op"] == "rope":
        t, per = case["n"] * case["per"], case["per"]
        big = 1.0 + 7.0 * (torch.rand(hd, device="cuda", generator=_gen(seed, 9)) < 0.01).float()
        # the projections' rows: query and gate of each head side by side where gated
        st["qraw"] = _normal((t, H, (2 if case["gated"] else 1) * hd), 1.0, seed, 2)
        st["qraw"][:, :, :hd] *= big
        st["kraw"], st["vraw"] = _normal((t, KH, hd), 1.0, seed, 3) * big, _normal((t, KH, hd), 1.0, seed, 4)
        st["qn"], st["kn"] = _normal(hd, 0.1, seed, 5), _normal(hd, 0.1, seed, 6)
        st["freq"], st["mag"] = _freq(case), 0.1 * math.log(case["factor"]) + 1.0
        st["seq"] = _ints([s for s in range(case["n"]) for _ in range(per)])
        st["pos"] = _ints([x - per + i for x in lens for i in range(per)])
        st["q"] = torch.empty((t, H, hd), device="cuda")
    elif case["op"] == "attn":
        _spoil(case, st, lens)
        n = case["n"]
        st["q"] = _normal((n, H, hd), 1.3, seed, 2)
        st["qraw"] = _normal((n, H, (2 if case["gated"] else 1) * hd), 1.0, seed, 3)
        order = list(range(n))
        random.Random(n).shuffle(order)
        st["seq"], st["max_len"] = _ints(order), max(lens)
        st["out"] = torch.empty((n, H, hd), device="cuda")
        st["scratch"] = torch.zeros(64 << 20, dtype=torch.uint8, device="cuda")
        st["mag"], st["freq"] = 1.0, None
    elif case["op"] == "fork":
        n, each = case["n"], case["each"]
        per = 1 if case["share"] else max(_pages_of(lens, page))
        st.update(_pool(case, seed, lens, n * each * per + 3, n * each))
        st["src"] = _ints([s for s in range(n) for _ in range(each)])
        st["dst"] = _ints(list(range(n, n + n * each)))
    else:
        st.update(_pool(case, seed, lens, 7, 0, spans=_group(case)))
        st["groups"] = [(_ints(g), _ints([lens[s] for s in g]), sum(_pages_of([lens[s] for s in g], page)))
                        for g in _group(case)]
    return st


# ---------------------------------------------------------------- the plain forms
def _rotate(x, cos, sin, rot, style):
    if rot == 0:
        return x
    a, rest = x[..., :rot], x[..., rot:]
    if style == "half":
        u, v = a[..., :rot // 2], a[..., rot // 2:]
        return torch.cat((u * cos - v * sin, v * cos + u * sin, rest), -1)
    u, v = a[..., 0::2], a[..., 1::2]
    return torch.cat((torch.stack((u * cos - v * sin, v * cos + u * sin), -1).flatten(-2), rest), -1)


def _norm(x, w):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (1.0 + w)


def _plain_rope(st):
    c, page = st["case"], st["case"]["page"]
    ang = st["pos"].to(F64)[:, None] * st["freq"].to(F64)
    cos, sin = (torch.cos(ang) * st["mag"]).float()[:, None], (torch.sin(ang) * st["mag"]).float()[:, None]
    st["q"].copy_(_rotate(_norm(st["qraw"][:, :, :c["hd"]], st["qn"]), cos, sin, c["rot"], c["style"]))
    k = _rotate(_norm(st["kraw"], st["kn"]), cos, sin, c["rot"], c["style"])
    pos = st["pos"].long()
    at, slot = st["table"][st["seq"].long(), pos // page].long(), pos % page
    layer = st["data"][:, st["layer"]]
    layer[at, 0, :, slot] = k.to(layer.dtype)
    layer[at, 1, :, slot] = st["vraw"].to(layer.dtype)
    return {"q": st["q"], "data": st["data"]}


def _plain_attn(st):
    c, page = st["case"], st["case"]["page"]
    n, H, KH, hd, seq = c["n"], c["H"], c["KH"], c["hd"], st["seq"].long()
    P = max(1, (st["max_len"] + page - 1) // page)
    at = st["table"][seq, :P].long().clamp(min=0)
    kv = st["data"][:, st["layer"]][at]                                  # [n, P, 2, KH, page, hd]
    kv = kv.permute(2, 0, 3, 1, 4, 5).reshape(2, n, KH, P * page, hd).float()
    seen = torch.arange(P * page, device="cuda") < st["lens"][seq][:, None]
    v = torch.where(seen[:, None, :, None], kv[1], torch.zeros((), device="cuda"))
    s = st["q"].view(n, KH, H // KH, hd) @ kv[0].transpose(2, 3).contiguous() * (1.0 / math.sqrt(hd))
    s = torch.where(seen[:, None, None], s, torch.full((), -math.inf, device="cuda"))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    o = (p @ v) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    o = o.reshape(n, H, hd)
    if c["gated"]:
        o = o / (1.0 + torch.exp(-st["qraw"][:, :, hd:]))
    st["out"].copy_(o)
    return {"out": st["out"]}


def _in_use(st, seq):
    """The table rows of sequences and which of their entries are in use."""
    page, rows = st["case"]["page"], st["table"][seq].long()
    count = (st["lens"][seq].long() + page - 1) // page
    return rows, torch.arange(rows.shape[1], device="cuda") < count[:, None]


def _plain_free(st, seq):
    rows, live = _in_use(st, seq)
    st["refs"].index_add_(0, rows.clamp(min=0).flatten(), -live.flatten().int())
    st["lens"][seq], st["table"][seq] = 0, -1


def _plain_take(st, need):
    """The page ids of sum(need) new pages, the lowest free ones first; refs set."""
    free = torch.argsort((st["refs"] > 0).int(), stable=True)[:need]
    st["refs"][free] = 1
    return free


def _plain_fork(st):
    c, page = st["case"], st["case"]["page"]
    src, dst = st["src"].long(), st["dst"].long()
    _plain_free(st, dst)
    rows, live = _in_use(st, src)
    length = st["lens"][src].long()
    if c["share"]:
        full, part = length // page, length % page
        new_entry = torch.arange(rows.shape[1], device="cuda") == torch.where(part > 0, full, -1)[:, None]
    else:
        new_entry = live
    old, kept = rows[new_entry], live & ~new_entry
    new = _plain_take(st, old.numel())
    st["refs"].index_add_(0, rows.clamp(min=0).flatten(), kept.flatten().int())
    rows[new_entry] = new
    st["table"][dst], st["lens"][dst] = rows.int(), length.int()
    held = (length[:, None] - torch.arange(rows.shape[1], device="cuda") * page).clamp(max=page)[new_entry]
    sel = (torch.arange(page, device="cuda") < held[:, None])[:, None, None, None, :, None]
    st["data"][new] = torch.where(sel, st["data"][old], st["data"][new])
    return {k: st[k] for k in ("table", "lens", "refs", "data")}


def _plain_churn(st):
    seq, count, _ = st["groups"][st["turn"]]
    st["turn"] ^= 1
    seq, page = seq.long(), st["case"]["page"]
    _plain_free(st, seq)
    used = st["refs"] > 0
    ids, live = torch.arange(used.numel(), device="cuda"), used.sum()
    hole, mover = (~used & (ids < live)).nonzero()[:, 0], (used & (ids >= live)).nonzero()[:, 0]
    st["data"][hole] = st["data"][mover]
    ids[mover] = hole
    st["table"].copy_(torch.where(st["table"] >= 0, ids[st["table"].long().clamp(min=0)].int(), st["table"]))
    st["refs"][hole], st["refs"][mover] = st["refs"][mover], 0
    st["lens"][seq] = count
    _, entry = _in_use(st, seq)
    rows = st["table"][seq]
    rows[entry] = _plain_take(st, int(entry.sum())).int()
    st["table"][seq] = rows
    return {k: st[k] for k in ("table", "lens", "refs", "data")}


# ---------------------------------------------------------------- the library
_lib = None


def _library():
    global _lib
    if _lib is None:
        here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen3.c_amd", "__init__.py")
        spec = importlib.util.spec_from_file_location("qwen3_c_amd", here)
        mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
        _lib = mod.Lib().init()
    return _lib


def _handles(st):
    """The descriptions of the pool and the heads, made at the first pass on a state and kept
    beside it as a program keeps them."""
    if "pool" not in st:
        c, lib = st["case"], _library()
        st["pool"] = lib.pages(
            *(st[k].data_ptr() for k in ("data", "table", "lens", "refs", "used", "state", "work")), CODES[c["dtype"]],
            c["layers"], c["KH"], c["hd"], c["page"], st["refs"].numel(), st["lens"].numel(), st["table"].shape[1])
        if c["op"] in ("rope", "attn"):
            addr = lambda k: st[k].data_ptr() if st.get(k) is not None else None  # noqa: E731
            wide = 2 if c["gated"] else 1
            st["heads"] = lib.heads(
                H=c["H"], rot=c["rot"] if c["op"] == "rope" else 0, interleaved=c["style"] == "interleaved",
                q_row=c["H"] * wide * c["hd"], q_head=wide * c["hd"], kv_row=c["KH"] * c["hd"], eps=EPS,
                rope_mag=st["mag"], scale=1.0 / math.sqrt(c["hd"]), qn=addr("qn"), kn=addr("kn"), freq=addr("freq"))
    return _library(), st["pool"], st.get("heads")


def _stream():
    """torch's current stream, on which the inputs were made and the outputs are read; its default one by
    the name that is not NULL (the library's own stream): hipStreamLegacy."""
    return torch.cuda.current_stream().cuda_stream or 1


def _own_rope(st):
    lib, pool, heads = _handles(st)
    lib.qk_rope_paged_dev(pool, heads, st["layer"], st["qraw"].data_ptr(), st["kraw"].data_ptr(), st["vraw"].data_ptr(),
                          st["seq"].data_ptr(), st["pos"].data_ptr(), st["seq"].numel(), st["q"].data_ptr(), _stream())
    return {"q": st["q"], "data": st["data"]}


def _own_attn(st):
    lib, pool, heads = _handles(st)
    c = st["case"]
    gate = st["qraw"].data_ptr() + 4 * c["hd"] if c["gated"] else None
    lib.attn_paged_dev(pool, heads, st["layer"], st["q"].data_ptr(), gate, st["seq"].data_ptr(), None, c["n"],
                       st["max_len"], st["out"].data_ptr(), st["scratch"].data_ptr(), st["scratch"].numel(), _stream())
    return {"out": st["out"]}


def _own_fork(st):
    lib, pool, _ = _handles(st)
    n, stream = st["dst"].numel(), _stream()
    lib.pages_free(pool, st["dst"].data_ptr(), n, stream)
    lib.pages_fork(pool, st["src"].data_ptr(), st["dst"].data_ptr(), n, st["case"]["share"], stream)
    return {k: st[k] for k in ("table", "lens", "refs", "data")}


def _own_churn(st):
    lib, pool, _ = _handles(st)
    seq, count, _ = st["groups"][st["turn"]]
    st["turn"] ^= 1
    stream = _stream()
    lib.pages_free(pool, seq.data_ptr(), seq.numel(), stream)
    lib.pages_compact(pool, stream)
    lib.pages_append(pool, seq.data_ptr(), count.data_ptr(), seq.numel(), stream)
    return {k: st[k] for k in ("table", "lens", "refs", "data")}


def run(st):
    op = st["case"]["op"]
    if own:
        return {"rope": _own_rope, "attn": _own_attn, "fork": _own_fork, "churn": _own_churn}[op](st)
    return {"rope": _plain_rope, "attn": _plain_attn, "fork": _plain_fork, "churn": _plain_churn}[op](st)


# ---------------------------------------------------------------- 64 bits, from the definitions
def _exact_rope(st):
    c, hd, page = st["case"], st["case"]["hd"], st["case"]["page"]
    hr = c["rot"] // 2
    first = torch.arange(hr, device="cuda") * (1 if c["style"] == "half" else 2)
    second = first + (hr if c["style"] == "half" else 1)
    turn = torch.polar(torch.full((), st["mag"], dtype=F64, device="cuda"), st["pos"].to(F64)[:, None] * st["freq"].to(F64))

    def head(x, w):
        x = x.to(F64)
        x = x / (x.square().sum(-1, keepdim=True) / hd + EPS).sqrt() * (w.to(F64) + 1)
        z = torch.complex(x[..., first], x[..., second]) * turn[:, None]
        x[..., first], x[..., second] = z.real, z.imag
        return x

    data = st["data"].to(F64)
    k = head(st["kraw"], st["kn"])
    table, seq, pos = st["table"].cpu(), st["seq"].cpu(), st["pos"].cpu()
    where = torch.tensor([int(table[s, p // page]) * page + p % page for s, p in zip(seq.tolist(), pos.tolist())],
                         device="cuda")
    for which, x in ((0, k), (1, st["vraw"].to(F64))):
        for h in range(c["KH"]):
            plane = data[:, st["layer"], which, h].reshape(-1, hd)
            plane[where] = x[:, h]
            data[:, st["layer"], which, h] = plane.view(-1, page, hd)
    return {"q": head(st["qraw"][..., :hd], st["qn"]), "data": data}


def _exact_attn(st):
    c, page = st["case"], st["case"]["page"]
    H, KH, hd = c["H"], c["KH"], c["hd"]
    out = torch.zeros((c["n"], H, hd), dtype=F64, device="cuda")
    lens, table = st["lens"].tolist(), st["table"].long()
    for r, s in enumerate(st["seq"].tolist()):
        if not lens[s]:
            continue
        pg = st["data"][table[s, :(lens[s] + page - 1) // page], st["layer"]]
        for h in range(KH):
            k, v = (pg[:, i, h].reshape(-1, hd)[:lens[s]].to(F64) for i in (0, 1))
            q = st["q"][r, h * (H // KH):(h + 1) * (H // KH)].to(F64)
            w = torch.softmax(q @ k.T / math.sqrt(hd), -1)
            out[r, h * (H // KH):(h + 1) * (H // KH)] = w @ v
    return {"out": out * torch.sigmoid(st["qraw"][..., hd:].to(F64)) if c["gated"] else out}


def _exact_pages(st):
    """Where every page's rows end up, by plain lists."""
    c, page = st["case"], st["case"]["page"]
    table, lens, refs = st["table"].tolist(), st["lens"].tolist(), st["refs"].tolist()
    data = st["data"].to(F64)
    if c["op"] == "fork":
        for s, d in zip(st["src"].tolist(), st["dst"].tolist()):
            for j in range((lens[s] + page - 1) // page):
                held = min(page, lens[s] - j * page)
                if c["share"] and held == page:
                    continue
                new = refs.index(0)
                refs[new] = 1
                data[new, :, :, :, :held] = data[table[s][j], :, :, :, :held]
        return {"table": None, "lens": None, "refs": None, "data": data}
    for s in st["groups"][0][0].tolist():
        for p in table[s]:
            if p >= 0:
                refs[p] -= 1
    live = sum(r > 0 for r in refs)
    holes = [p for p in range(live) if not refs[p]]
    movers = [p for p in range(live, len(refs)) if refs[p]]
    if holes:
        data[torch.tensor(holes, device="cuda")] = data[torch.tensor(movers, device="cuda")]
    return {"table": None, "lens": None, "refs": None, "data": data}


def exact(case, seed):
    st = prepare(case, seed)
    return {"rope": _exact_rope, "attn": _exact_attn, "fork": _exact_pages, "churn": _exact_pages}[case["op"]](st)
