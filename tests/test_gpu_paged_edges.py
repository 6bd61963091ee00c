"""Edges of the paged key-value cache on the GPU: steps that run out of pages, rows over bad pages,
infinities at odd head dims, calls at once, the largest batches."""
import importlib.util
import math
import os

import numpy as np
import pytest
import torch

import _layers
import _paged
import _util
from _paged import BF16, F16, F32, Pool, addr, ints
from test_gpu_paged import Attn, sync

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mod():
    return _util.load_product()


@pytest.fixture(scope="module")
def dev(torch_dev):
    return torch_dev


# ---------------------------------------------------------------- an append that is refused
H, KH, HD, PAGE = 4, 2, 16, 4


class Step:
    """A decode step of two layers (append, then rows at their sequences' last positions) over a pool."""

    def __init__(self, mod, lib, dev, pool, n):
        self.lib, self.dev, self.pool, self.n = lib, dev, pool, n
        self.att = Attn(mod, lib, dev, pool, H, False)
        self.heads = mod.Lib.heads(H=H, rot=0, interleaved=0, q_row=H * HD, q_head=HD, kv_row=KH * HD, eps=1e-6,
                                   rope_mag=1.0, scale=0.25)
        self.seq = ints([-1] * n, dev)
        self.x = [torch.zeros(n, h * HD, device=dev) for h in (H, KH, KH)]
        self.qo, self.out = (torch.zeros(2, n, H, HD, device=dev) for _ in range(2))

    def run(self, st):
        lib, c, n = self.lib, self.pool.c, self.n
        lib.pages_append(c, addr(self.seq), None, n, st)
        for l in range(2):
            lib.qk_rope_paged_dev(c, self.heads, l, *(addr(t) for t in self.x), addr(self.seq), None, n,
                                  addr(self.qo[l]), st)
            lib.attn_paged_dev(c, self.att.heads, l, addr(self.qo[l]), None, addr(self.seq), None, n, 0,
                               addr(self.out[l]), addr(self.att.work), self.att.work.numel(), st)

    def capture(self):
        self.run(None)   # of no sequences: the kernels are loaded before the capture
        sync(self.lib)
        side, self.graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph, stream=side):
            self.run(torch.cuda.current_stream().cuda_stream)

    def replay(self, seq, seed):
        g = torch.Generator().manual_seed(seed)
        for t in self.x:
            t.copy_(torch.randn(t.shape, generator=g))
        self.seq.copy_(ints(seq, self.dev))
        self.qo.fill_(5.0)
        torch.cuda.synchronize()
        self.graph.replay()
        torch.cuda.synchronize()
        return self.lib.pages_status(self.pool.c)


def written(pool, step, data, seq, lens):
    """`data` with the rows of the step at the last positions of its sequences."""
    for r, s in enumerate(seq):
        if s >= 0:
            at = lens[s] - 1
            pg = int(pool.table[s, at // PAGE])
            for kv in (0, 1):
                data[pg, :, kv, :, at % PAGE] = step.x[1 + kv][r].view(KH, HD).to(data.dtype)
    return data


@pytest.mark.parametrize("why", ["shared", "own", "row"])
def test_refused_append_writes_nothing(mod, lib, dev, why):
    """A captured step whose append is refused (no free page, the last page of two branches shared or
    not; a table row that is full) changes no page, for any sequence of the batch; the same graph goes
    on once pages are free or the full sequence is out of the batch."""
    full = why == "row"
    pool = Pool(mod, lib, dev, F32, 2, KH, HD, PAGE, 20 if full else {"shared": 6, "own": 8}[why], 4,
                2 if full else 6, seed=3)
    pool.place([8, 0 if why == "shared" else 6 if full else 8, 0 if full else 12, 0])
    if why == "shared":
        lib.pages_fork(pool.c, addr(a := ints([0], dev)), addr(b := ints([1], dev)), 1, True)
        sync(lib)
        assert pool.table[0, :2].tolist() == pool.table[1, :2].tolist()
    step = Step(mod, lib, dev, pool, 3)
    step.capture()
    lens, data, table = pool.lens.tolist(), pool.data.clone(), pool.table.clone()
    for t in range(2):
        free, err = step.replay([1, -1, 0], t)
        assert err == (2 if full else 1) | 16 and pool.lens.tolist() == lens
        assert torch.equal(pool.data, data) and torch.equal(pool.table, table)
        assert bool((step.qo == 5.0).all())
    if full:
        seq = [1, -1, -1]
    else:
        seq = [1, -1, 0]
        lib.pages_free(pool.c, addr(x := ints([2], dev)), 1)
        sync(lib)
    for t in range(2, 4):
        before = pool.data.clone()
        free, err = step.replay(seq, t)
        for s in seq:
            lens[s] += s >= 0
        if not full:
            lens[2] = 0
        assert err == 0 and pool.lens.tolist() == lens
        assert torch.equal(pool.data, written(pool, step, before, seq, lens)), t
        for r, s in enumerate(seq):
            assert torch.equal(step.qo[1, r].view(-1), step.x[0][r] if s >= 0 else torch.full((H * HD,), 5.0, device=dev))
    n = [lens[s] for s in seq]
    step.att.check(torch.where(torch.tensor(seq)[:, None, None] < 0, 77.0, step.out[1].cpu()), step.qo[1].cpu(),
                   torch.zeros(3, step.att.heads.q_row), seq, n, layer=1)


def test_refused_append_is_forgotten(mod, lib, dev):
    """What a refused append leaves holds only until its sequence grows, is freed or forked into, also where
    the length comes to the same again; a count of 0 asks for no place; an unnamed sequence is not held up."""
    pool = Pool(mod, lib, dev, F32, 2, KH, HD, PAGE, 9, 6, 6, seed=3)
    step = Step(mod, lib, dev, pool, 1)
    keep = []

    def call(f, *lists):
        t = [ints(v, dev) if isinstance(v, list) else v for v in lists]
        keep.extend(t)
        torch.cuda.synchronize()
        f(pool.c, *(addr(v) if torch.is_tensor(v) else v for v in t))

    def writes(s):
        """Whether a row without d_pos of sequence s goes to its last position, and the error bits."""
        before = pool.data.clone()
        g = torch.Generator().manual_seed(len(keep))
        for t in step.x:
            t.copy_(torch.randn(t.shape, generator=g))
        keep.append(q := ints([s], dev))
        torch.cuda.synchronize()
        for l in range(2):
            lib.qk_rope_paged_dev(pool.c, step.heads, l, *(addr(t) for t in step.x), addr(q), None, 1, addr(step.qo[l]))
        sync(lib)
        err = lib.pages_status(pool.c)[1]
        if torch.equal(pool.data, before):
            return False, err
        assert torch.equal(pool.data, written(pool, step, before, [s], pool.lens.tolist()))
        return True, err

    call(lib.pages_append, [0, 1, 2], [8, 8, 8], 3)             # 6 of 9 pages
    for s in range(3):
        assert writes(s) == (True, 0)
    call(lib.pages_append, [0, 1, 3], [4, 0, 40], 3)            # refused: 0 and 3, the row of 3 too short
    assert lib.pages_status(pool.c) == (3, 2)
    assert writes(0) == (False, 16) and writes(1) == (True, 0) and writes(2) == (True, 0) and writes(3) == (False, 16)
    call(lib.pages_append, [0], [0], 1)                         # grows by nothing: still without its place
    assert writes(0) == (False, 16)
    call(lib.pages_free, [0], 1)
    call(lib.pages_append, [0], [8], 1)                         # the same length again
    assert writes(0) == (True, 0)
    call(lib.pages_append, [2, 9], [1, 1], 2)                   # refused for the other's sake
    assert lib.pages_status(pool.c)[1] == 4
    assert writes(2) == (False, 16)
    call(lib.pages_free, [2], 1)
    call(lib.pages_fork, [0], [2], 1, 1)                        # as long as before, by a fork
    assert writes(2) == (True, 0)
    call(lib.pages_append, [1], [-1], 1)
    assert lib.pages_status(pool.c)[1] == 4 and writes(1) == (False, 16)
    call(lib.pages_append, [1], [1], 1)
    assert writes(1) == (True, 0)
    call(lib.pages_append, [1, 1], None, 2)
    assert lib.pages_status(pool.c)[1] == 8 and writes(1) == (False, 16)
    lib.pages_init(pool.c)
    call(lib.pages_append, [1], [9], 1)
    assert writes(1) == (True, 0)


def test_refused_append_layer_block(mod, lib, gen, dev):
    """The layer block of a step without pages gives 0 and keeps the cache."""
    D, rot, gs = 256, 16, 128
    W = _layers.GqaWeights(gen, gen.stream(0x9F00, 1), D, 4, 2, 64, rot, gs)
    tq, tk, tv, to = (m.upload(lib) for m in (W.q, W.k, W.v, W.o))
    pool = Pool(mod, lib, dev, BF16, 1, 2, 64, 4, 4, 2, 4, seed=2)
    freq = torch.tensor([float(np.float32(float(W.theta) ** (-2.0 * j / rot))) for j in range(rot // 2)], device=dev)
    heads = mod.Lib.heads(H=4, rot=rot, interleaved=0, q_row=8 * 64, q_head=2 * 64, kv_row=2 * 64, eps=1e-6,
                          rope_mag=1.0, scale=1.0 / math.sqrt(64), freq=addr(freq))
    x = torch.from_numpy(np.concatenate([gen.normal(D, 0x9F10 + t) for t in range(2)])).to(dev)
    seq, cnt = ints([0, 1], dev), ints([8, 7], dev)

    def go(count):
        out = torch.full((2, D), 4.0, device=dev)
        torch.cuda.synchronize()
        lib.pages_append(pool.c, addr(seq), addr(count), 2)
        lib.gqa_paged_dev(pool.c, heads, 0, addr(x), tq, tk, tv, to, addr(seq), None, 2, 9, addr(out))
        sync(lib)
        return out, lib.pages_status(pool.c)[1]

    out, err = go(cnt)
    assert err == 0 and bool(out.any(1).all())
    data = pool.data.clone()
    out, err = go(None)
    assert err == 1 | 16 and not bool(out.any()) and torch.equal(pool.data, data)


# ---------------------------------------------------------------- infinities at head dims of their own
@pytest.mark.parametrize("hint", [0, 200], ids=["shares", "whole"])
@pytest.mark.parametrize("hd", [8, 72, 80, 176])
@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "f16", "f32"])
def test_attn_minus_infinity(mod, lib, dev, dtype, hd, hint):
    """A key with -inf in a column where the queries are positive has no weight, whatever the head dim
    is padded to; +inf there and NaN give NaN, for its heads alone; an infinity of V stays in its column."""
    KH, page, length = 2, 16, 200
    pool = Pool(mod, lib, dev, dtype, 1, KH, hd, page, 5 * 13 + 1, 5, 14, seed=4)
    pool.place([length] * 5)
    a = Attn(mod, lib, dev, pool, 4, True, seed=3)
    q, raw = a.rows(5)
    q[:3, :, :4], q[0, 2:, hd - 1] = q[:3, :, :4].abs(), q[0, 2:, hd - 1].abs()
    t, inf = pool.table.long(), float("inf")
    clean = a.run(q, raw, list(range(5)), max_len=hint)
    a.check(clean, q, raw, list(range(5)), [length] * 5)
    pool.data[t[0, 3], 0, 0, 0, 5, 0] = -inf         # the first column of the key
    pool.data[t[0, 12], 0, 0, 0, 2, 3] = -inf
    pool.data[t[0, 7], 0, 0, 1, 9, hd - 1] = -inf    # the last
    pool.data[t[1, 0], 0, 0, 1, 0, 1] = inf
    pool.data[t[2, 1], 0, 0, 0, 1, 2] = float("nan")
    pool.data[t[3, 2], 0, 1, 1, 3, hd - 2] = inf
    torch.cuda.synchronize()
    got = a.run(q, raw, list(range(5)), max_len=hint)
    K, V = (pool.rows(0, 0, length, i) for i in (0, 1))
    fin = torch.isfinite(K).all(-1)
    want = torch.cat([_paged.attn(q[0, 2 * h:2 * h + 2], K[h:h + 1, fin[h]], V[h:h + 1, fin[h]], a.scale,
                                  a.gate_of(raw, 0)[2 * h:2 * h + 2])[0] for h in range(KH)])
    assert torch.allclose(got[0].double(), want, rtol=1e-5, atol=1e-5)
    assert bool(torch.isnan(got[1, 2:]).all()) and bool(torch.isnan(got[2, :2]).all())
    assert bool((got[3, 2:, hd - 2] == inf).all())
    rest = clean.clone()
    rest[0], rest[1, 2:], rest[2, :2], rest[3, 2:, hd - 2] = got[0], got[1, 2:], got[2, :2], got[3, 2:, hd - 2]
    assert torch.allclose(got, rest, rtol=2e-5, atol=2e-5, equal_nan=True)


# ---------------------------------------------------------------- calls at once
def test_status_loses_no_bits(mod, lib, dev):
    """Error bits that an attention call on another stream sets while the status is read are in this
    reading or in the next."""
    pool = Pool(mod, lib, dev, BF16, 1, 1, 64, 16, 64, 2, 32, seed=4)
    pool.place([400, 100])
    a, b = (Attn(mod, lib, dev, pool, 4, False, seed=i) for i in (1, 2))
    q = a.rows(1)[0].to(dev)
    out = [torch.zeros(1, 4, 64, device=dev) for _ in range(2)]
    none, one, far = ints([-2], dev), ints([0], dev), ints([4000], dev)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for t in range(400):
        lib.attn_paged_dev(pool.c, a.heads, 0, addr(q), None, addr(none), None, 1, 0, addr(out[0]), addr(a.work),
                           a.work.numel())                                             # bit 4
        lib.sync()
        for i in range(t % 20 + 1):   # the last one sets bit 16, later from turn to turn
            lib.attn_paged_dev(pool.c, b.heads, 0, addr(q), None, addr(one), addr(far) if i == t % 20 else None, 1, 0,
                               addr(out[1]), addr(b.work), b.work.numel(), side.cuda_stream)
        first = lib.pages_status(pool.c)[1]
        torch.cuda.synchronize()
        second = lib.pages_status(pool.c)[1]
        assert first | second == 4 | 16, (t, first, second)
    assert lib.pages_status(pool.c)[1] == 0


# ---------------------------------------------------------------- rows over pages that are none
@pytest.mark.parametrize("hint", [0, 150, 40], ids=["shares", "whole", "whole-short"])
@pytest.mark.parametrize("hd", [64, 80])
@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "f16", "f32"])
def test_attn_all_pages_bad(mod, lib, dev, dtype, hd, hint):
    """A row all of whose table entries are no pages sees nothing and gives 0, a short one and one in
    parts; rows whose first or last keys alone are there see those; a row all of whose keys have -inf
    scores has no softmax (NaN), as the formula has it, also where its other pages are bad."""
    KH, page = 2, 16
    lens = [5, 3000, 40, 3000, 3000, 16, 3000, 3000]
    pool = Pool(mod, lib, dev, dtype, 1, KH, hd, page, 5 * 188 + 10, 8, 190, seed=4)
    pool.place(lens)
    a = Attn(mod, lib, dev, pool, 4, True, seed=3)
    q, raw = a.rows(8)
    q[5:7, :, 1] = q[5:7, :, 1].abs() + 0.1
    t = pool.table
    t[0, 0] = -1
    t[1, :188] = pool.n_pages
    t[2, 0], t[2, 2] = -5, 2 ** 31 - 1               # the middle page alone
    t[3, :100] = -1                                  # parts of no keys before those that have some
    t[4, 3:188] = -1                                 # and behind them
    for s, n in ((5, 1), (6, 188)):
        pool.data[t[s, :n].long(), 0, 0, :, :, 1] = -float("inf")
    t[6, 20:120] = -1
    torch.cuda.synchronize()
    got = a.run(q, raw, list(range(8)), max_len=hint)
    assert lib.pages_status(pool.c)[1] == 32
    assert bool((got[:2] == 0.0).all()), got[:2]
    for s, keys in ((2, range(16, 32)), (3, range(1600, 3000)), (4, range(48))):
        held = [p for j, p in enumerate(t[s, :-(-lens[s] // page)].tolist()) if 0 <= p < pool.n_pages]
        x = pool.data[held, 0].cpu().double().permute(1, 2, 0, 3, 4).reshape(2, KH, -1, hd)[:, :, :len(keys)]
        want = _paged.attn(q[s], x[0], x[1], a.scale, a.gate_of(raw, s))[0]
        assert torch.allclose(got[s].double(), want, rtol=1e-5, atol=1e-5), s
    assert bool(torch.isnan(got[5:7]).all())
    a.check(got[7:], q[7:], raw[7:], [7], [lens[7]])


# ---------------------------------------------------------------- the largest batches
def test_projection_of_many_rows(lib, gen, dev):
    """2^20 rows, what a call of the paged cache may have, through a projection of 1024 columns: rows at
    both ends and about every border of its pieces against a small call's.  The two may sum in another
    order: 1024 products of 24 bits, 6 sqrt(1024) half steps of the largest output."""
    I, O, S = 1024, 48, 1 << 20
    q, sz = gen.fmt6(O, I, 128, 0xA100)
    t = lib.tensor(q, sz, 6, I, O, 128)
    x = torch.randn(S, I, device=dev)
    most = (2 ** 31 - 1) // (3 * I)
    rows = [0, 1, 2 ** 18 - 1, 2 ** 18, 2 ** 19, most - 1, most, most + 1, S - 2, S - 1]
    few = x[rows].contiguous()
    y, z = torch.full((S, O), float("nan"), device=dev), torch.zeros(len(rows), O, device=dev)
    torch.cuda.synchronize()
    lib.gemv_dev(t, addr(x), addr(y), S)
    lib.gemv_dev(t, addr(few), addr(z), len(rows))
    lib.sync()
    assert not bool(torch.isnan(y).any())
    assert bool(((y[rows] - z).abs() <= 2 * 6 * 32 * _paged.U * z.abs().max()).all())


def test_layer_block_of_many_rows(mod, lib, gen, dev):
    """A layer block of 2^20 rows, 2^32 values of context: the few rows that have a position, from the
    first to the last, come out as in a call of their own (the projections' sums in another order), the
    others give 0."""
    D, nh, hd, n = 128, 16, 256, 1 << 20
    tq, tk, tv, to = (lib.tensor(*gen.fmt6(O, I, 128, 0xA200 + i), 6, I, O, 128)
                      for i, (O, I) in enumerate(((nh * hd, D), (hd, D), (hd, D), (64, nh * hd))))
    pool = Pool(mod, lib, dev, F32, 1, 1, hd, 4, 12, 3, 4, seed=2)
    pool.place([13, 9, 16])
    heads = mod.Lib.heads(H=nh, rot=0, interleaved=0, q_row=nh * hd, q_head=hd, kv_row=hd, eps=1e-6, rope_mag=1.0,
                          scale=1.0 / math.sqrt(hd))
    rows = [0, 3, 4095, n // 2, n - 2, n - 1]
    few_seq, few_pos = ints([0, 1, 2, 0, 1, 2], dev), ints([12, 3, 15, 5, 8, 0], dev)
    seq, pos = torch.full((n,), -1, dtype=torch.int32, device=dev), torch.zeros(n, dtype=torch.int32, device=dev)
    seq[rows], pos[rows] = few_seq, few_pos
    x = torch.randn(n, D, device=dev)
    few = x[rows].contiguous()
    out, want = torch.full((n, 64), 3.0, device=dev), torch.full((6, 64), 3.0, device=dev)
    for hint in (0, 16):
        out.fill_(3.0)
        torch.cuda.synchronize()
        lib.gqa_paged_dev(pool.c, heads, 0, addr(x), tq, tk, tv, to, addr(seq), addr(pos), n, hint, addr(out))
        sync(lib)
        lib.gqa_paged_dev(pool.c, heads, 0, addr(few), tq, tk, tv, to, addr(few_seq), addr(few_pos), 6, hint, addr(want))
        sync(lib)
        assert lib.pages_status(pool.c)[1] == 0
        for r in range(6):
            assert _util.maxrel_scaled(out[rows[r]].cpu().numpy(), want[r].cpu().numpy()) <= 1e-3, r
        out[rows] = 0.0
        assert not bool(out.any())


# ---------------------------------------------------------------- calls in a program's stream order
def _operators():
    spec = importlib.util.spec_from_file_location("operators", os.path.join(_util.ROOT, "perf", "operators.py"))
    ops = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ops)
    return ops


@pytest.mark.parametrize("side", [False, True], ids=["default", "side"])
def test_calls_follow_the_current_stream(dev, side):
    """Inputs made on torch's current stream, the library's calls, outputs copied on that stream, with no
    wait between them: as with every step waited for.  Work that takes a while goes ahead of the inputs."""
    ops, case = _operators(), dict(name="", op="attn", n=16, len=900, ragged=True, H=8, KH=2, hd=64, rot=64, style="half",
                                   dtype="bf16", page=16, layers=1, gated=True)
    ops.own = True
    big = torch.randn(4096, 4096, device=dev)
    st, other = ops.prepare(case, 1), ops.prepare(case, 2)
    torch.cuda.synchronize()
    want, late = (ops.run(s)["out"].clone() for s in (st, other))
    torch.cuda.synchronize()
    ops._library().sync()
    want, late = ops.run(st)["out"].cpu(), ops.run(other)["out"].cpu()
    q1, q2 = st["q"].clone(), other["q"].clone()
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream() if side else torch.cuda.current_stream()):
        for i in range(6):
            for s, q in ((st, q1), (other, q2)):
                s["q"].zero_()
                s["out"].fill_(-3.0)
            for _ in range(4):
                torch.mm(big, big)
            st["q"].copy_(q1)
            other["q"].copy_(q2)
            a = ops.run(st)["out"].clone()
            b = ops.run(other)["out"].clone()
            st["out"].fill_(9.0)
            assert torch.equal(a.cpu(), want) and torch.equal(b.cpu(), late), i


def test_default_stream_by_its_name(mod, lib, gen, dev):
    """hipStreamLegacy (1), the name of the default stream that is not NULL: a projection, the layer block,
    the bookkeeping, the status and the wait, behind torch's work on that stream and ahead of its copies."""
    D, legacy = 256, 1
    W = _layers.GqaWeights(gen, gen.stream(0xA300, 1), D, 4, 2, 64, 16, 128)
    tq, tk, tv, to = (m.upload(lib) for m in (W.q, W.k, W.v, W.o))
    heads = mod.Lib.heads(H=4, rot=0, interleaved=0, q_row=8 * 64, q_head=2 * 64, kv_row=2 * 64, eps=1e-6,
                          rope_mag=1.0, scale=0.125)
    big, xs, lists = torch.randn(4096, 4096, device=dev), torch.randn(5, D, device=dev), ints([0, 1, 2, 3, 4], dev)
    got = []
    for stream in (None, legacy):
        pool = Pool(mod, lib, dev, BF16, 1, 2, 64, 4, 12, 5, 4, seed=2)
        x, seq, out, y = torch.zeros_like(xs), ints([-1] * 5, dev), torch.zeros(5, D, device=dev), torch.zeros(5, 512, device=dev)
        torch.cuda.synchronize()
        for _ in range(8):
            torch.mm(big, big)
        x.copy_(xs)
        seq.copy_(lists)
        if stream is None:
            torch.cuda.synchronize()
        lib.pages_append(pool.c, addr(seq), None, 5, stream)
        lib.gqa_paged_dev(pool.c, heads, 0, addr(x), tq, tk, tv, to, addr(seq), None, 5, 1, addr(out), stream)
        lib.gemv_dev(tq, addr(x), addr(y), 5, stream)
        if stream is None:
            lib.sync()
        copies = out.clone(), y.clone(), pool.lens.clone()
        assert lib.pages_status(pool.c, stream) == (7, 0)
        lib.sync(stream)
        got.append(copies)
    assert bool(got[0][0].any(1).all()) and all(torch.equal(a, b) for a, b in zip(*got))
