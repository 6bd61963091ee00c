"""The paged key-value cache on the GPU: its bookkeeping against a model in plain Python (equal,
copied rows bit for bit), norms / rotation / page writes and attention against 64-bit forms on
the CPU, the layer block against the CPU oracle, and what a captured decode step leaves.

Tolerances are of fp32 arithmetic (derived beside each bound), plus half a step of the pages'
type where a value is rounded to it.
"""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import _layers
import _paged
import _util
from _paged import BF16, F16, F32, NAMES, TORCH, U, Model, Pool, addr, ints

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mod():
    return _util.load_product()


@pytest.fixture(scope="module")
def dev(torch_dev):
    return torch_dev


def sync(lib):
    torch.cuda.synchronize()
    lib.sync()


# ---------------------------------------------------------------- bookkeeping
@pytest.mark.parametrize("dtype,layers,KH,hd,page,seed", [
    (BF16, 2, 2, 64, 16, 1), (F32, 1, 1, 8, 1, 2), (F16, 3, 2, 72, 5, 3), (F32, 1, 3, 256, 8, 4), (BF16, 1, 1, 16, 33, 5),
], ids=lambda v: str(v))
def test_random_life(mod, lib, dev, dtype, layers, KH, hd, page, seed):
    """Appends, forks, frees and compactions in random order, failing ones among them: tables,
    lengths, counts, bitmap and every page's contents after each."""
    n_pages, n_seqs, max_pages = 75, 12, 14
    pool = Pool(mod, lib, dev, dtype, layers, KH, hd, page, n_pages, n_seqs, max_pages, seed)
    m = Model(pool)
    m.check(pool, lib, "init")
    rng = np.random.default_rng(seed)
    for step in range(60):
        op = rng.choice(["append", "append", "append", "fork", "fork", "free", "compact"])
        if op == "append":
            k = int(rng.integers(1, 6))
            s = rng.choice(n_seqs, k, replace=rng.random() < 0.1).tolist()
            s = [-1 if rng.random() < 0.15 else x for x in s]
            c = None if rng.random() < 0.4 else rng.integers(0, 4 * page + 1, k).tolist()
            if rng.random() < 0.05:
                s[0] = n_seqs
            done = m.append(s, c)
            lib.pages_append(pool.c, addr(a := ints(s, dev)), addr(b := ints(c, dev) if c else None), k)
        elif op == "fork":
            k = int(rng.integers(1, 5))
            empty = [s for s in range(n_seqs) if not m.lens[s]]
            a = rng.choice(n_seqs, k).tolist()
            b = (empty * k)[:k] if empty and rng.random() < 0.2 else rng.permutation(empty + [-1] * k)[:k].tolist()
            if rng.random() < 0.1:
                a[-1] = -1
            share = bool(rng.random() < 0.6)
            done = m.fork(a, b, share)
            lib.pages_fork(pool.c, addr(a := ints(a, dev)), addr(b := ints(b, dev)), k, share)
        elif op == "free":
            s = rng.choice(n_seqs, int(rng.integers(1, 4))).tolist() + [-1]
            m.free(s)
            done = True
            lib.pages_free(pool.c, addr(a := ints(s, dev)), len(s))
        else:
            m.compact()
            done = True
            lib.pages_compact(pool.c)
        m.check(pool, lib, (step, op, done))


def test_bookkeeping_refusals(mod, lib, dev):
    """Calls the device cannot carry out leave the pool as it was and set their bit; counts of
    zero, empty lists and padding do nothing."""
    pool = Pool(mod, lib, dev, BF16, 1, 1, 8, 4, 6, 4, 4)
    m = Model(pool)

    def app(s, c=None):
        m.append(s, c)
        lib.pages_append(pool.c, addr(a := ints(s, dev)), addr(b := None if c is None else ints(c, dev)), len(s))
        m.check(pool, lib, (s, c))

    app([0, 1], [9, 4])          # 3 + 1 pages of 6
    app([2], [0])
    app([-1, -1])
    app([2, 3], [5, 5])          # needs 4: out of pages
    app([0], [8])                # 17 positions in a row of 16
    app([0], [2 ** 31 - 1])
    app([1, 1])                  # twice
    app([4])                     # no such sequence
    app([-2])
    app([2], [-1])
    app([0, 2], [7, 4])          # the last two pages, the row full to its end
    app([1])                     # none left
    for a, b, share in (([0], [0], 1), ([0], [1], 1), ([0], [3], 0), ([0, 1], [3, 3], 1), ([5], [3], 1), ([0], [9], 1),
                        ([-1], [3], 1), ([0], [-1], 0), ([3], [3], 1)):
        m.fork(a, b, share)
        lib.pages_fork(pool.c, addr(x := ints(a, dev)), addr(y := ints(b, dev)), len(a), share)
        m.check(pool, lib, (a, b, share))
    m.fork([0], [3], True)       # full pages only: needs none
    lib.pages_fork(pool.c, addr(x := ints([0], dev)), addr(y := ints([3], dev)), 1, True)
    m.check(pool, lib, "share all")
    for s in ([0, 0], [7], [-3], [3, -1, 1], [3]):
        m.free(s)
        lib.pages_free(pool.c, addr(x := ints(s, dev)), len(s))
        m.check(pool, lib, s)
    L, p = lib.L, C.byref(pool.c)
    one = ints([0], dev)
    assert L.coli_hip_pages_append(p, None, None, 0, None) == 1
    assert L.coli_hip_pages_append(p, None, None, 1, None) == 0
    assert L.coli_hip_pages_append(p, addr(one), None, -1, None) == 0
    assert L.coli_hip_pages_append(p, addr(one), None, 4097, None) == 0
    assert L.coli_hip_pages_fork(p, addr(one), None, 1, 1, None) == 0
    assert L.coli_hip_pages_free(p, None, 2, None) == 0
    assert L.coli_hip_pages_free(p, addr(one), 4097, None) == 0
    m.check(pool, lib, "after refusals")


def test_large_pool(mod, lib, dev):
    """Pages past one round of the free-page search (32768 pages), thousands of new pages in a
    call, a call of 4096 sequences, and compaction across the words' borders."""
    n_pages, n_seqs, max_pages = 100_003, 4100, 40_000
    pool = Pool(mod, lib, dev, F16, 1, 1, 8, 1, n_pages, n_seqs, 40_000, fill=False)
    pool.data.view(torch.int16).copy_(torch.randint(-30000, 30000, pool.data.shape, dtype=torch.int16))
    torch.cuda.synchronize()
    m = Model(pool)

    def app(s, c):
        assert m.append(s, c)
        lib.pages_append(pool.c, addr(a := ints(s, dev)), addr(b := ints(c, dev)), len(s))
        m.check(pool, lib, "append")

    def free(s):
        m.free(s)
        lib.pages_free(pool.c, addr(a := ints(s, dev)), len(s))
        lib.sync()

    app([0, 1, 2], [39_000, 1, 31_000])
    app(list(range(3, 4099)), [i % 3 for i in range(4096)])
    free([1, 0] + list(range(10, 3000, 2)))
    m.check(pool, lib, "free")
    assert m.fork([2], [0], False)
    lib.pages_fork(pool.c, addr(a := ints([2], dev)), addr(b := ints([0], dev)), 1, False)
    m.check(pool, lib, "copy")
    free([2])
    m.compact()
    lib.pages_compact(pool.c)
    m.check(pool, lib, "compact")
    m.compact()
    lib.pages_compact(pool.c)
    m.check(pool, lib, "compact again")
    assert not m.append([2], [40_001])
    lib.pages_append(pool.c, addr(a := ints([2], dev)), addr(b := ints([40_001], dev)), 1)
    m.check(pool, lib, "row too long")
    app([2, 1], [40_000, 9_000])   # to nearly the last page


# ---------------------------------------------------------------- norms, rotation, pages
ROPE = [   # dtype, H, KH, hd, rot, interleaved, norms, gated, page, n, far
    (BF16, 16, 2, 256, 64, 0, True, True, 16, 3, 0), (F16, 32, 8, 128, 128, 1, True, False, 32, 19, 0),
    (F32, 8, 8, 64, 64, 0, False, False, 7, 65, 0), (BF16, 3, 1, 80, 40, 1, True, True, 1, 5, 0),
    (F32, 5, 5, 8, 8, 1, True, False, 4, 9, 0), (F16, 4, 2, 72, 0, 0, True, True, 16, 7, 0),
    (F32, 2, 1, 248, 2, 0, True, False, 128, 4, 0), (F32, 4, 2, 64, 32, 0, True, False, 4096, 4, 1_000_000_000),
    (BF16, 4, 1, 176, 64, 1, True, True, 64, 200, 3_000_000),
]


@pytest.mark.parametrize("dtype,H,KH,hd,rot,inter,norms,gated,page,n,far", ROPE, ids=lambda v: str(v))
def test_qk_rope(mod, lib, dev, dtype, H, KH, hd, rot, inter, norms, gated, page, n, far):
    """Queries out, keys and values in their slots and nothing else changed; rows of no sequence
    skipped.  Far positions: a row whose table is long enough, one page of it real.

    Bound of a rotated value: the sum of squares is a tree (10 roundings: 5 in the root), mean,
    eps, root, quotient, (1 + w) and two products 8; the angle is rounded once at up to half a
    turn (pi U), its sine and cosine to 2 ulp (4 U), the magnitude 1, two products and a sum 3:
    24 U of |u| + |v| covers it."""
    layers, layer, n_seqs = 2, 1, n + 2
    rng = np.random.default_rng(n * 7 + hd)
    need = far // page + 1 if far else 6
    pool = Pool(mod, lib, dev, dtype, layers, KH, hd, page, 6 * n_seqs, n_seqs, need, seed=hd)
    if far:
        lens = [0] * n_seqs
        table = torch.full((n_seqs, need), -1, dtype=torch.int32)
        pos = [far - 13 * i for i in range(n)]
        for s in range(n):
            lens[s] = pos[s] + 1
            table[s, pos[s] // page] = 5 * n_seqs - s
        pool.table.copy_(table)
        pool.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        torch.cuda.synchronize()
    else:
        lens = [int(x) for x in rng.integers(1, 5 * page + 1, n)]
        pool.place(lens)
        pos = [int(rng.integers(0, x)) for x in lens]
    seq = list(range(n))
    if n > 3:
        seq[2] = -1
    wide = 2 if gated else 1
    g = torch.Generator().manual_seed(n)
    pad = 3   # columns between rows: strides are not the sizes
    q = torch.randn(n, H * wide * hd + pad, generator=g) * 2
    k, v = torch.randn(n, KH * hd + pad, generator=g), torch.randn(n, KH * hd + pad, generator=g)
    qn, kn = (torch.randn(hd, generator=g) * 0.2, torch.randn(hd, generator=g) * 0.2) if norms else (None, None)
    freq = (torch.tensor(1e6, dtype=torch.float64) ** (-torch.arange(rot // 2).double() * 2 / max(rot, 1))).float()
    mag = 1.25 if inter else 1.0
    d = [t.to(dev) if t is not None else None for t in (q, k, v, qn, kn, freq)]
    out = torch.full((n, H, hd), 123.0, device=dev)
    heads = mod.Lib.heads(H=H, rot=rot, interleaved=inter, q_row=q.shape[1], q_head=wide * hd, kv_row=k.shape[1],
                          eps=1e-6, rope_mag=mag, scale=1.0, qn=addr(d[3]), kn=addr(d[4]), freq=addr(d[5]))
    before = pool.data.cpu().clone()
    sq, ps = ints(seq, dev), ints(pos, dev)
    torch.cuda.synchronize()
    lib.qk_rope_paged_dev(pool.c, heads, layer, addr(d[0]), addr(d[1]), addr(d[2]), addr(sq), addr(ps), n, addr(out))
    sync(lib)
    assert lib.pages_status(pool.c)[1] == 0
    q3 = q[:, :H * wide * hd].view(n, H, wide * hd)[..., :hd]
    k3, v3 = k[:, :KH * hd].view(n, KH, hd), v[:, :KH * hd].view(n, KH, hd)
    pt = torch.tensor(pos)
    rq, sizeq = _paged.rope64(_paged.norm64(q3, qn, 1e-6), pt, freq, rot, inter, mag)
    rk, sizek = _paged.rope64(_paged.norm64(k3, kn, 1e-6), pt, freq, rot, inter, mag)
    got, want, table = out.cpu().double(), before, pool.table.cpu()
    after = pool.data.cpu()
    for r in range(n):
        if seq[r] == -1:
            assert bool((got[r] == 123.0).all())
            continue
        assert bool(((got[r] - rq[r]).abs() <= 24 * U * sizeq[r] + 1e-37).all()), (r, pos[r])
        pg, slot = int(table[r, pos[r] // page]), pos[r] % page
        gk, tiny = after[pg, layer, 0, :, slot].double(), (2.0 ** -25 if dtype == F16 else 1e-37)
        half = torch.finfo(TORCH[dtype]).eps / 2 if dtype != F32 else 0.0
        b = 24 * U * sizek[r]
        assert bool(((gk - rk[r]).abs() <= b + half * (rk[r].abs() + b) + tiny).all()), (r, pos[r])
        assert torch.equal(after[pg, layer, 1, :, slot], v3[r].to(TORCH[dtype]))
        want[pg, layer, :, :, slot] = after[pg, layer, :, :, slot]
    assert torch.equal(after, want)   # nothing but those slots


def test_qk_rope_last_position_and_refusals(mod, lib, dev):
    """d_pos NULL is each sequence's last position; rows past the end, of an empty or no sequence,
    or over a bad table entry write nothing and set their bit."""
    H, KH, hd, page, n = 2, 1, 16, 4, 6
    pool = Pool(mod, lib, dev, F32, 1, KH, hd, page, 30, n, 4, seed=3)
    lens = [3, 8, 9, 0, 16, 1]
    pool.place(lens)
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(n, h * hd, generator=g).to(dev) for h in (H, KH, KH))
    heads = mod.Lib.heads(H=H, rot=0, interleaved=0, q_row=H * hd, q_head=hd, kv_row=KH * hd, eps=1e-6, rope_mag=1.0,
                          scale=1.0)

    def go(seq, pos, layer=0):
        out = torch.full((len(seq), H, hd), 5.0, device=dev)
        before = pool.data.clone()
        s, p = ints(seq, dev), None if pos is None else ints(pos, dev)
        torch.cuda.synchronize()
        lib.qk_rope_paged_dev(pool.c, heads, layer, addr(q), addr(k), addr(v), addr(s), addr(p), len(seq), addr(out))
        sync(lib)
        return out, before, lib.pages_status(pool.c)[1]

    out, before, err = go([0, 1, 2, 4, 5], None)
    assert err == 0 and torch.equal(out.view(5, -1), q[:5])
    for r, s in enumerate([0, 1, 2, 4, 5]):
        at = lens[s] - 1
        before[int(pool.table[s, at // page]), 0, 0, 0, at % page] = k[r]
        before[int(pool.table[s, at // page]), 0, 1, 0, at % page] = v[r]
    assert torch.equal(pool.data, before)
    for seq, pos, bit in (([3], None, 0), ([0], [3], 16), ([0], [2 ** 31 - 1], 16), ([0], [-1], 0), ([0], [-2], 4),
                          ([6], None, 4), ([-2], None, 4), ([-1], None, 0)):
        out, before, err = go(seq, pos)
        assert err == bit and torch.equal(pool.data, before) and bool((out == 5.0).all()), (seq, pos, err)
    pool.table[1, 1] = 30
    out, before, err = go([1], None)
    assert err == 32 and torch.equal(pool.data, before)
    L, P, hp = lib.L, C.byref(pool.c), C.byref(heads)
    s = ints([0], dev)
    for a in ((P, hp, 1, addr(q), addr(k), addr(v), addr(s), None, 1, addr(out), None),
              (P, hp, -1, addr(q), addr(k), addr(v), addr(s), None, 1, addr(out), None),
              (P, hp, 0, None, addr(k), addr(v), addr(s), None, 1, addr(out), None),
              (P, hp, 0, addr(q), addr(k), addr(v), None, None, 1, addr(out), None),
              (P, hp, 0, addr(q), addr(k), addr(v), addr(s), None, -1, addr(out), None),
              (P, None, 0, addr(q), addr(k), addr(v), addr(s), None, 1, addr(out), None)):
        assert L.coli_hip_qk_rope_paged(*a) == 0
    assert L.coli_hip_qk_rope_paged(P, hp, 0, None, None, None, None, None, 0, None, None) == 1


# ---------------------------------------------------------------- attention
class Attn:
    """Rows over a pool: run through the library, held to the 64-bit form."""

    def __init__(self, mod, lib, dev, pool, H, gated, scale=None, seed=0):
        self.mod, self.lib, self.dev, self.pool, self.H, self.gated = mod, lib, dev, pool, H, gated
        self.scale = scale if scale is not None else 1.0 / math.sqrt(pool.hd)
        wide = 2 if gated else 1
        self.heads = mod.Lib.heads(H=H, rot=0, interleaved=0, q_row=H * wide * pool.hd + 5, q_head=wide * pool.hd,
                                   kv_row=pool.KH * pool.hd, eps=1e-6, rope_mag=1.0, scale=self.scale)
        self.g = torch.Generator().manual_seed(seed)
        self.work = torch.zeros(lib.attn_paged_work(pool.c, self.heads), dtype=torch.uint8, device=dev)

    def rows(self, n, sigma=1.0):
        return (torch.randn(n, self.H, self.pool.hd, generator=self.g) * sigma,
                torch.randn(n, self.heads.q_row, generator=self.g))

    def run(self, q, raw, seq, pos=None, max_len=0, layer=0, stream=None, out=None):
        n, dev = len(seq), self.dev
        dq, dr, s = q.to(dev), raw.to(dev), ints(seq, dev)
        p = None if pos is None else ints(pos, dev)
        out = torch.full((n, self.H, self.pool.hd), 77.0, device=dev) if out is None else out
        torch.cuda.synchronize()
        gate = addr(dr) + 4 * self.pool.hd if self.gated else None
        self.lib.attn_paged_dev(self.pool.c, self.heads, layer, addr(dq), gate, addr(s), addr(p), n, max_len, addr(out),
                                addr(self.work), self.work.numel(), stream)
        sync(self.lib)
        return out.cpu()

    def gate_of(self, raw, r):
        hd = self.pool.hd
        return raw[r, :2 * self.H * hd].view(self.H, 2 * hd)[:, hd:] if self.gated else None

    def check(self, got, q, raw, seq, counts, layer=0):
        """Every row within the elementwise bound; and the rows' relative errors, in the mean, no
        more than 4 times those of the same formula in fp32 (or 2^-20, where that is luckier): the
        order of the sums differs, their precision must not."""
        off = off32 = rows = 0.0
        for r, s in enumerate(seq):
            if s < 0:
                assert bool((got[r] == 77.0).all()), r
                continue
            n = counts[r]
            K, V = (self.pool.rows(layer, s, n, i) for i in (0, 1))
            ref, size, big = _paged.attn(q[r], K, V, self.scale, self.gate_of(raw, r))
            b = _paged.attn_bound(size, big, self.pool.hd, n)
            d = (got[r].double() - ref).abs()
            assert bool((d <= b).all()), (r, s, n, float((d / b).max()))
            low = _paged.attn(q[r], K, V, self.scale, self.gate_of(raw, r), dtype=torch.float32)[0].double()
            if n:
                sq = float((ref * ref).sum())
                off, off32 = off + float((d * d).sum()) / sq, off32 + float(((low - ref) ** 2).sum()) / sq
                rows += 1
        if rows:
            e, e32 = math.sqrt(off / rows), math.sqrt(off32 / rows)
            print(f"{NAMES[self.pool.dtype]} H {self.H} KH {self.pool.KH} hd {self.pool.hd}: {e:.2e}, in fp32 {e32:.2e}",
                  flush=True)
            assert e <= max(4 * e32, 2.0 ** -20), (e, e32)


def lens_for(page):
    return sorted({0, 1, 2, page - 1, page, page + 1, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 255, 256, 257, 300, 511,
                   513, 700})


ATTN = [   # dtype, H, KH, hd, page, gated
    (BF16, 16, 2, 256, 16, True), (F16, 16, 2, 256, 16, False), (F32, 16, 2, 256, 16, True),
    (BF16, 32, 8, 128, 32, False), (F16, 8, 8, 64, 1, True), (F32, 5, 1, 128, 5, False), (BF16, 12, 4, 80, 20, True),
    (F16, 40, 8, 112, 64, False), (BF16, 16, 1, 176, 7, False), (F32, 3, 3, 8, 16, True), (F16, 17, 1, 72, 16, False),
    (BF16, 64, 2, 64, 128, False), (F32, 33, 1, 248, 24, False), (BF16, 2, 2, 24, 4096, False),
]


@pytest.mark.parametrize("dtype,H,KH,hd,page,gated", ATTN, ids=lambda v: str(v))
def test_attn_lengths(mod, lib, dev, dtype, H, KH, hd, page, gated):
    """Lengths around the pages' and tiles' borders, rows in no order, padding among them; slots
    past the ends hold NaN and infinities."""
    lens = lens_for(page)
    n = len(lens)
    P = -(-max(lens) // page)
    pool = Pool(mod, lib, dev, dtype, 2, KH, hd, page, sum(-(-x // page) for x in lens) + 3, n + 1, P + 1, seed=H)
    pool.place(lens, seed=hd)
    for s, x in enumerate(lens):
        if x % page:
            pool.data[pool.table[s, x // page].long(), :, 0, :, x % page:] = float("nan")
            pool.data[pool.table[s, x // page].long(), :, 1, :, x % page:] = float("inf") if s % 2 else float("nan")
    torch.cuda.synchronize()
    a = Attn(mod, lib, dev, pool, H, gated, seed=page)
    seq = np.random.default_rng(page).permutation(n).tolist()
    seq[3:3], seq[n:n] = [-1], [-1]
    q, raw = a.rows(len(seq))
    for max_len in (0, max(lens)):
        got = a.run(q, raw, seq, max_len=max_len, layer=1)
        a.check(got, q, raw, seq, [0 if s < 0 else lens[s] for s in seq], layer=1)
        assert lib.pages_status(pool.c)[1] == 0
    one = lens.index(257)
    got1 = a.run(q[:1], raw[:1], [one], max_len=257, layer=1)   # a row alone
    a.check(got1, q[:1], raw[:1], [one], [257], layer=1)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_attn_positions(mod, lib, dev, dtype):
    """d_pos: several rows of one sequence, each over what it sees (a draft of tokens), nothing at
    -1; past the end: what is held, and the bit."""
    pool = Pool(mod, lib, dev, dtype, 1, 2, 64, 16, 60, 3, 30, seed=5)
    pool.place([400, 90, 0])
    a = Attn(mod, lib, dev, pool, 8, True, seed=1)
    seq = [0, 0, 0, 0, 1, 1, 1, 2, 0, 0]
    pos = [399, 398, 0, -1, 89, 15, 16, -1, 200, 127]
    q, raw = a.rows(len(seq))
    got = a.run(q, raw, seq, pos)
    a.check(got, q, raw, seq, [p + 1 for p in pos])
    assert bool((got[3] == 0).all()) and bool((got[7] == 0).all())
    assert lib.pages_status(pool.c)[1] == 0
    got = a.run(q[:3], raw[:3], [0, 1, 2], [400, 2 ** 31 - 1, 5])
    a.check(got, q[:3], raw[:3], [0, 1, 2], [400, 90, 0])
    assert lib.pages_status(pool.c)[1] == 16
    got = a.run(q[:3], raw[:3], [0, 3, -7], [-2, 0, 0])
    assert bool((got[0] == 0).all()) and bool((got[1:] == 77.0).all())
    assert lib.pages_status(pool.c)[1] == 4


@pytest.mark.parametrize("dtype,H,KH,hd,n,length", [(BF16, 16, 2, 256, 1, 40_001), (F16, 8, 1, 128, 2, 70_000),
                                                   (F32, 8, 4, 64, 1, 50_003)], ids=lambda v: str(v))
def test_attn_long(mod, lib, dev, dtype, H, KH, hd, n, length):
    """A long axis and few rows: the work of one row is split and joined.  One row is sharp (its
    largest weight far into the sequence), the hint of the length right, absent and wrong."""
    page = 16
    lens = [length - 1000 * i for i in range(n)]
    pool = Pool(mod, lib, dev, dtype, 1, KH, hd, page, sum(-(-x // page) for x in lens) + 1, n, -(-length // page) + 1,
                seed=9)
    pool.place(lens)
    a = Attn(mod, lib, dev, pool, H, False, seed=2)
    q, raw = a.rows(n)
    K = pool.rows(0, 0, lens[0], 0)
    q[0, 0] = (K[0, length // 2] * 3).float()
    first = None
    for hint in (length, 0, 100, 1 << 30):
        got = a.run(q, raw, list(range(n)), max_len=hint)
        if first is None:
            a.check(got, q, raw, list(range(n)), lens)
            first = got
        assert float((got.double() - first.double()).norm() / first.double().norm()) <= 2.0 ** -18
    again = a.run(q, raw, list(range(n)), max_len=length)
    assert torch.equal(again, first)   # the same call twice: the same bits


@pytest.mark.parametrize("dtype,KH,hd,n", [(BF16, 2, 64, 700), (F32, 1, 128, 300), (F16, 2, 256, 257), (BF16, 1, 8, 5000)],
                         ids=lambda v: str(v))
def test_attn_many_rows(mod, lib, dev, dtype, KH, hd, n):
    """More rows than a block has threads: drafts and short chats, rows of no sequence at both
    ends and between, several rows a sequence."""
    rng = np.random.default_rng(n)
    lens = [int(x) for x in rng.integers(0, 150, 40)]
    lens[7] = 2000
    pool = Pool(mod, lib, dev, dtype, 1, KH, hd, 16, sum(-(-x // 16) for x in lens) + 1, 40, 130, seed=3)
    pool.place(lens)
    a = Attn(mod, lib, dev, pool, 4 * KH, False, seed=1)
    seq = [int(x) for x in rng.integers(-1, 40, n)]
    seq[:3], seq[-2:] = [-1, -1, 7], [7, -1]
    pos = [int(rng.integers(-1, lens[s])) if s >= 0 else 5 for s in seq]
    q, raw = a.rows(n)
    got = a.run(q, raw, seq, pos)
    assert lib.pages_status(pool.c)[1] == 0
    check = sorted(set(range(0, n, max(1, n // 250))) | {0, 1, 2, n - 2, n - 1})
    pool.data = pool.data.cpu()
    a.check(got[check], q[check], raw[check], [seq[i] for i in check], [pos[i] + 1 for i in check])
    rest = [i for i in range(n) if seq[i] < 0 or pos[i] < 0]
    assert bool((got[rest] == torch.tensor([77.0 if seq[i] < 0 else 0.0 for i in rest])[:, None, None]).all())


@pytest.mark.parametrize("dtype,H,KH,hd,n,page", [
    (BF16, 32, 8, 128, 80, 16), (F16, 8, 8, 64, 70, 5), (F32, 16, 8, 128, 64, 32), (BF16, 18, 1, 80, 600, 16),
    (F16, 4, 4, 8, 130, 1), (F32, 6, 2, 72, 270, 16), (F16, 24, 4, 112, 128, 64), (BF16, 7, 1, 64, 513, 24),
], ids=lambda v: str(v))
def test_attn_short_and_many(mod, lib, dev, dtype, H, KH, hd, n, page):
    """Many short rows: a length as long as the hint, one
    far past it, none at all, rows of no sequence; the same rows without a hint agree, and where an
    infinity or NaN is seen they agree on that."""
    rng = np.random.default_rng(n)
    lens = [int(x) for x in rng.integers(1, 90, 30)] + [0, 1, 1000, 3500]
    pool = Pool(mod, lib, dev, dtype, 1, KH, hd, page, sum(-(-x // page) for x in lens) + 1, len(lens),
                -(-3500 // page), seed=3)
    pool.place(lens)
    a = Attn(mod, lib, dev, pool, H, n % 2 == 0, seed=1)
    seq = [int(x) for x in rng.integers(-1, len(lens), n)]
    seq[:4], seq[-2:] = [-1, 33, 32, 31], [30, -1]
    counts = [lens[s] if s >= 0 else 0 for s in seq]
    q, raw = a.rows(n)
    got = a.run(q, raw, seq, max_len=1000)
    assert lib.pages_status(pool.c)[1] == 0
    check = sorted(set(range(0, n, max(1, n // 60))) | {0, 1, 2, 3, n - 2, n - 1})
    a.check(got[check], q[check], raw[check], [seq[i] for i in check], [counts[i] for i in check])
    free = a.run(q, raw, seq)
    assert torch.allclose(got, free, rtol=1e-4, atol=1e-5)
    assert torch.equal(got, a.run(q, raw, seq, max_len=1000))
    for s, kv, x in ((3, 1, float("inf")), (33, 0, float("nan")), (32, 1, float("-inf"))):
        pool.data[pool.table[s, 0].long(), 0, kv, 0, 0, 5] = x
    torch.cuda.synchronize()
    got, free = a.run(q, raw, seq, max_len=1000), a.run(q, raw, seq)
    assert not bool(torch.isfinite(got).all())
    assert torch.allclose(got, free, rtol=1e-4, atol=1e-5, equal_nan=True)


@pytest.mark.parametrize("dtype,H,KH,hd,n,page,hints", [
    (BF16, 32, 8, 128, 90, 16, (5, 40, 200, 0)), (BF16, 16, 2, 256, 300, 16, (40, 90, 200)),
    (F16, 8, 8, 64, 150, 5, (30, 60, 500)), (F32, 16, 8, 128, 80, 32, (9, 33, 150)), (BF16, 18, 1, 80, 600, 16, (8, 50, 64)),
    (F16, 4, 4, 8, 300, 1, (16, 33, 300)), (F32, 6, 2, 72, 270, 16, (12, 70)), (F16, 24, 4, 112, 140, 64, (64, 150)),
    (BF16, 7, 1, 64, 1100, 24, (32, 33, 1000)), (F32, 5, 5, 256, 60, 8, (20, 140)), (F16, 40, 2, 200, 280, 16, (31, 99)),
    (F32, 8, 8, 48, 140, 16, (16, 17, 300)), (BF16, 2, 1, 136, 3, 16, (1, 30)), (F16, 20, 1, 128, 1, 16, (1, 90)),
], ids=lambda v: str(v))
def test_attn_whole_rows(mod, lib, dev, dtype, H, KH, hd, n, page, hints):
    """Hints small enough that a block of one wave or of four has a (row, kv head) to itself: lengths
    up to the hint, none, one far past it; rows of no sequence; infinities and NaN."""
    for hint in hints:
        rng = np.random.default_rng(1000 * n + hint)
        top = max(hint, 1)
        lens = [int(x) for x in rng.integers(0, top + 1, 20)] + [top, 0, 1, max(1, top - 1), 1500]
        pool = Pool(mod, lib, dev, dtype, 2, KH, hd, page, sum(-(-x // page) for x in lens) + 1, len(lens),
                    -(-1500 // page), seed=hint)
        pool.place(lens)
        a = Attn(mod, lib, dev, pool, H, n % 2 == 0, seed=1)
        seq = [int(x) for x in rng.integers(-1, len(lens), n)]
        seq[0] = 20
        if n > 8:
            seq[1:5], seq[-2:] = [-1, 24, 21, 22], [23, -1]
        counts = [lens[s] if s >= 0 else 0 for s in seq]
        q, raw = a.rows(n)
        got = a.run(q, raw, seq, max_len=hint)
        assert lib.pages_status(pool.c)[1] == 0
        check = sorted(set(range(0, n, max(1, n // 40))) | set(range(min(n, 5))) | {n - 1, max(0, n - 2)})
        a.check(got[check], q[check], raw[check], [seq[i] for i in check], [counts[i] for i in check])
        none = [i for i in range(n) if seq[i] < 0]
        assert bool((got[none] == 77.0).all())
        assert torch.equal(got, a.run(q, raw, seq, max_len=hint))
        if hint:
            few = min(n, 3)
            some = a.run(q[:few].contiguous(), raw[:few].contiguous(), seq[:few], max_len=hint)
            assert torch.allclose(some, got[:few], rtol=1e-4, atol=1e-5)
        for s, kv, x in ((20, 1, float("inf")), (22, 0, float("nan"))):
            if lens[s]:
                pool.data[pool.table[s, 0].long(), 0, kv, 0, 0, 5] = x
        torch.cuda.synchronize()
        got, free = a.run(q, raw, seq, max_len=hint), a.run(q, raw, seq)
        assert not bool(torch.isfinite(got[0]).all())
        assert torch.allclose(got, free, rtol=1e-4, atol=1e-5, equal_nan=True)


def test_offsets_past_32_bits(mod, lib, dev):
    """A pool of 6.5 GB whose sequence lies at its far end: rows written, attended, copied there and
    moved down from there."""
    H, KH, hd, page, layers, n_pages = 8, 2, 256, 16, 10, 20_000
    pool = Pool(mod, lib, dev, BF16, layers, KH, hd, page, n_pages, 3, 8, fill=False)
    far = [n_pages - 1, n_pages - 7, n_pages - 3]
    pool.table[0, :3] = ints(far, dev)
    refs = np.zeros(n_pages, np.int32)
    refs[far] = 1
    refs[5] = 1   # page 5 is another's: the copies go around it
    pool.table[2, 0], pool.lens[2] = 5, 3
    pool.refs.copy_(torch.from_numpy(refs))
    pool.used.copy_(torch.from_numpy(_paged.bitmap(refs)))
    n = 40
    pool.lens[0] = n
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(n, h * hd, generator=g) for h in (H, KH, KH))
    d = [t.to(dev) for t in (q, k, v)]
    heads = mod.Lib.heads(H=H, rot=0, interleaved=0, q_row=H * hd, q_head=hd, kv_row=KH * hd, eps=1e-6, rope_mag=1.0,
                          scale=1.0 / 16)
    out, s, p = torch.zeros(n, H, hd, device=dev), ints([0] * n, dev), ints(range(n), dev)
    torch.cuda.synchronize()
    lib.qk_rope_paged_dev(pool.c, heads, layers - 1, *(addr(t) for t in d), addr(s), addr(p), n, addr(out))
    sync(lib)
    K, V = (pool.rows(layers - 1, 0, n, i) for i in (0, 1))
    assert torch.equal(K, k.view(n, KH, hd).bfloat16().double().transpose(0, 1))
    assert torch.equal(V, v.view(n, KH, hd).bfloat16().double().transpose(0, 1))
    a = Attn(mod, lib, dev, pool, H, False)
    qq, raw = a.rows(2)
    a.check(a.run(qq, raw, [0, 0], [n - 1, 17], layer=layers - 1), qq, raw, [0, 0], [n, 18], layer=layers - 1)
    lib.pages_fork(pool.c, addr(x := ints([0], dev)), addr(y := ints([1], dev)), 1, False)
    lib.sync()
    assert pool.table[1, :4].tolist() == [0, 1, 2, -1]
    assert torch.equal(pool.rows(layers - 1, 1, n, 0), K) and torch.equal(pool.rows(layers - 1, 1, n, 1), V)
    lib.pages_compact(pool.c)
    lib.sync()   # 7 pages: those past them, in order, into 3, 4 and 6; page 5 stays
    assert pool.table[0, :4].tolist() == [6, 3, 4, -1] and pool.table[2, 0] == 5
    assert torch.equal(pool.rows(layers - 1, 0, n, 0), K) and torch.equal(pool.rows(layers - 1, 0, n, 1), V)
    assert lib.pages_status(pool.c) == (n_pages - 7, 0)


def test_attn_rows_in_several_launches(mod, lib, dev):
    """Table rows of 2^30 positions: four rows' units fill a launch's counter, ten rows take three
    launches over one workspace."""
    pool = Pool(mod, lib, dev, F32, 1, 16, 8, 4096, 12, 10, 1 << 18, seed=3)
    lens = [4097, 1, 300, 0, 4096, 64, 65, 5000, 129, 4000]
    pool.place(lens)
    a = Attn(mod, lib, dev, pool, 16, True, seed=1)
    q, raw = a.rows(10)
    got = a.run(q, raw, list(range(10)))
    a.check(got, q, raw, list(range(10)), lens)
    assert lib.pages_status(pool.c)[1] == 0


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "f16", "f32"])
def test_attn_extremes(mod, lib, dev, dtype):
    """Scores far apart, all alike, queries of 0, large and tiny; tiny and large values; keys in
    rising and falling order of their scores (the running maximum moves at every key)."""
    H, KH, hd, page, length = 8, 2, 64, 16, 333
    pool = Pool(mod, lib, dev, dtype, 1, KH, hd, page, 6 * 21 + 2, 6, 22, seed=4)
    pool.place([length] * 6)
    base = torch.randn(hd, generator=torch.Generator().manual_seed(1))
    top = torch.finfo(TORCH[dtype]).max
    for s in range(6):
        pg = pool.table[s, :21].long()
        sl = torch.arange(21 * page, device=dev)
        K = pool.data[pg, 0, 0]
        if s == 0:      # rising
            K = (base.to(dev)[None, None, :] * (sl.view(21, 1, page, 1) / length)).expand(21, KH, page, hd)
        elif s == 1:    # falling
            K = (base.to(dev)[None, None, :] * (1 - sl.view(21, 1, page, 1) / length)).expand(21, KH, page, hd)
        elif s == 2:    # all alike
            K = base.to(dev).expand(21, KH, page, hd)
        pool.data[pg, 0, 0] = K.to(TORCH[dtype])
        if s == 3:
            pool.data[pg, 0, 1] *= 1e-6 if dtype != F16 else 2.0 ** -10
        if s == 4:
            pool.data[pg, 0, 1] *= min(1e30, top / 64)
    torch.cuda.synchronize()
    a = Attn(mod, lib, dev, pool, H, False, seed=3)
    q, raw = a.rows(6)
    q[0], q[1] = base * 20, base * 20
    q[2, 0], q[2, 1] = 0, 1e-20
    q[3, 0] *= 30
    q[5, 0] *= 1e4
    got = a.run(q, raw, list(range(6)))
    a.check(got, q, raw, list(range(6)), [length] * 6)


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "f16", "f32"])
def test_attn_not_finite(mod, lib, dev, dtype):
    """Infinities and NaN in positions that a row sees go where the formula takes them, and no
    further: other heads, rows and columns keep their values."""
    H, KH, hd, page, length = 4, 2, 64, 16, 200
    pool = Pool(mod, lib, dev, dtype, 1, KH, hd, page, 5 * 13 + 1, 5, 14, seed=4)
    pool.place([length] * 5)
    a = Attn(mod, lib, dev, pool, H, False, seed=3)
    q, raw = a.rows(5)
    clean = a.run(q, raw, list(range(5)))
    t = pool.table.long()
    inf, nan = float("inf"), float("nan")
    pool.data[t[0, 3], 0, 1, 0, 5, 7] = inf     # V: column 7 of head 0's group
    pool.data[t[1, 3], 0, 1, 1, 5, 9] = nan
    pool.data[t[2, 3], 0, 0, 0, 5, 7] = nan     # K: every column of the group
    q[3, :2, 4] = q[3, :2, 4].abs()
    pool.data[t[3, 12], 0, 0, 0, 2, 4] = -inf   # K: a score of -inf: that key has no weight
    q[4, 2, 0] = nan
    torch.cuda.synchronize()
    got = a.run(q, raw, list(range(5)))
    K, V = pool.rows(0, 3, length, 0), pool.rows(0, 3, length, 1)
    want = _paged.attn(q[3], K, V, a.scale)[0].float()
    clean = clean.clone()
    for r, rows, col in ((0, slice(0, 2), 7), (1, slice(2, 4), 9)):
        bad = got[r, rows, col]
        assert bool((bad == inf).all() if r == 0 else torch.isnan(bad).all()), (r, bad)
        clean[r, rows, col] = bad
    for r, rows in ((2, slice(0, 2)), (4, slice(2, 3))):
        assert bool(torch.isnan(got[r, rows]).all())
        clean[r, rows] = got[r, rows]
    assert torch.allclose(got[3], want, rtol=1e-5, atol=1e-5)
    clean[3] = got[3]
    assert torch.allclose(got, clean, rtol=2e-5, atol=2e-5, equal_nan=True)


def test_attn_bad_pages(mod, lib, dev):
    """A table entry that is no page: its positions are left out, the bit is set, no fault."""
    pool = Pool(mod, lib, dev, BF16, 1, 1, 64, 16, 40, 2, 20, seed=4)
    pool.place([200, 100])
    a = Attn(mod, lib, dev, pool, 4, False)
    q, raw = a.rows(2)
    saved = int(pool.table[0, 5])
    K, V = pool.rows(0, 0, 200, 0), pool.rows(0, 0, 200, 1)
    keep = [i for i in range(200) if i // 16 != 5]
    want = _paged.attn(q[0], K[:, keep], V[:, keep], a.scale)[0].float()
    for bad in (-1, 40, 2 ** 31 - 1, -2 ** 31):
        pool.table[0, 5] = bad
        got = a.run(q, raw, [0, 1])
        assert lib.pages_status(pool.c)[1] == 32
        assert torch.allclose(got[0], want, rtol=1e-4, atol=1e-5)
    pool.table[0, 5] = saved


def test_attn_refusals(mod, lib, dev):
    pool = Pool(mod, lib, dev, BF16, 1, 1, 64, 16, 4, 2, 2)
    a = Attn(mod, lib, dev, pool, 4, False)
    L, P, h = lib.L, C.byref(pool.c), C.byref(a.heads)
    q, s, out = torch.zeros(1, 4, 64, device=dev), ints([0], dev), torch.zeros(1, 4, 64, device=dev)
    w, nb = addr(a.work), a.work.numel()
    ok = (P, h, 0, addr(q), None, addr(s), None, 1, 0, addr(out), w, nb, None)
    assert L.coli_hip_attn_paged(*ok) == 1
    for i, v in ((1, None), (2, 1), (2, -1), (3, None), (5, None), (7, -1), (7, (1 << 20) + 1), (9, None),
                 (9, addr(out) + 4), (10, None), (10, w + 8),
                 (11, nb - 1)):
        args = list(ok)
        args[i] = v
        assert L.coli_hip_attn_paged(*args) == 0, i
    assert L.coli_hip_attn_paged(P, h, 0, None, None, None, None, 0, 0, None, None, 0, None) == 1
    sync(lib)


@pytest.mark.parametrize("share", [True, False])
def test_fork_then_diverge(mod, lib, dev, share):
    """A run of them together: a prompt appended and written, forked, both grown by other tokens;
    each attends over its own history, the parent's rows untouched by the child's."""
    H, KH, hd, page, layers = 6, 2, 64, 8, 2
    pool = Pool(mod, lib, dev, BF16, layers, KH, hd, page, 40, 3, 12, seed=6)
    a = Attn(mod, lib, dev, pool, H, False)
    g = torch.Generator().manual_seed(4)
    freq = torch.tensor([1.0, 0.1, 0.01, 0.001], device=dev)
    heads = mod.Lib.heads(H=H, rot=8, interleaved=0, q_row=H * hd, q_head=hd, kv_row=KH * hd, eps=1e-6, rope_mag=1.0,
                          scale=a.scale, freq=addr(freq))
    hist = {0: [], 1: []}

    def write(seqs, pos):
        n = len(seqs)
        q, k, v = (torch.randn(n, h, hd, generator=g) for h in (H, KH, KH))
        out, s, p = torch.zeros(n, H, hd, device=dev), ints(seqs, dev), ints(pos, dev)
        d = [t.to(dev) for t in (q, k, v)]
        torch.cuda.synchronize()
        for layer in range(layers):
            lib.qk_rope_paged_dev(pool.c, heads, layer, *(addr(t) for t in d), addr(s), addr(p), n, addr(out))
        sync(lib)
        rk = _paged.rope64(k.double(), torch.tensor(pos), freq.cpu(), 8, 0, 1.0)[0]
        for r, x in enumerate(seqs):
            hist[x].append((rk[r], v[r]))
        return out

    def grow(seqs, n):
        lib.pages_append(pool.c, addr(s := ints(seqs, dev)), addr(c := ints([n] * len(seqs), dev)), len(seqs))
        lib.sync()

    grow([0], 21)
    write([0] * 21, list(range(21)))
    lib.pages_fork(pool.c, addr(x := ints([0], dev)), addr(y := ints([1], dev)), 1, share)
    lib.sync()
    hist[1] = list(hist[0])
    for t in range(12):
        grow([0, 1], 1)
        out = write([1, 0], [21 + t, 21 + t])
        got = a.run(out.cpu(), torch.zeros(2, a.heads.q_row), [1, 0], layer=1)
        for r, s in enumerate([1, 0]):
            K, V = (torch.stack([h[i] for h in hist[s]], 1).to(torch.bfloat16).double() for i in (0, 1))
            held, _ = pool.rows(1, s, 22 + t, 0), pool.rows(1, s, 22 + t, 1)
            # a key may be rounded to the other side of a tie: 2^-8 of it, and fp32 before that
            assert bool(((held - K).abs() <= 2.0 ** -7 * K.abs() + 1e-30).all())
            assert torch.equal(pool.rows(1, s, 22 + t, 1), V)
        a.check(got, out.cpu(), torch.zeros(2, a.heads.q_row), [1, 0], [22 + t] * 2, layer=1)
    assert lib.pages_status(pool.c)[1] == 0
    full = 21 // page
    shared = pool.table[0, :full].tolist() == pool.table[1, :full].tolist()
    assert shared == share and pool.table[0, full] != pool.table[1, full]


# ---------------------------------------------------------------- streams, graphs
def test_attn_two_streams(mod, lib, dev):
    """Calls at once on two streams, a workspace each, over one pool."""
    pool = Pool(mod, lib, dev, BF16, 1, 2, 128, 16, 700, 2, 400, seed=4)
    pool.place([5000, 4000])
    a, b = (Attn(mod, lib, dev, pool, 8, False, seed=i) for i in (1, 2))
    qa, raw = a.rows(2)
    qb, _ = b.rows(2)
    wa, wb = a.run(qa, raw, [0, 1]), b.run(qb, raw, [1, 0])
    s = [torch.cuda.Stream() for _ in range(2)]
    out = [torch.zeros(2, 8, 128, device=dev) for _ in range(2)]
    dq, sq = [qa.to(dev), qb.to(dev)], [ints([0, 1], dev), ints([1, 0], dev)]
    torch.cuda.synchronize()
    for _ in range(10):
        for i, x in enumerate((a, b)):
            lib.attn_paged_dev(pool.c, x.heads, 0, addr(dq[i]), None, addr(sq[i]), None, 2, 5000, addr(out[i]),
                               addr(x.work), x.work.numel(), s[i].cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(out[0].cpu(), wa) and torch.equal(out[1].cpu(), wb)


def test_captured_decode(mod, lib, dev):
    """A decode step (append, then norms / rotation / pages and attention of two layers) captured
    once and replayed, with eager work between: each replay against the same step run eagerly on
    a second pool, the sequences growing over page borders."""
    H, KH, hd, page, layers, n = 8, 2, 64, 4, 2, 4
    pools = [Pool(mod, lib, dev, BF16, layers, KH, hd, page, 64, n, 16, seed=8) for _ in range(3)]
    lens = [3, 0, 9, 4]
    for p in pools:
        lib.pages_append(p.c, addr(s := ints(range(n), dev)), addr(c := ints(lens, dev)), n)
        lib.sync()
    att = [Attn(mod, lib, dev, p, H, False) for p in pools]
    freq = torch.rand(16, device=dev)
    heads = mod.Lib.heads(H=H, rot=32, interleaved=0, q_row=H * hd, q_head=hd, kv_row=KH * hd, eps=1e-6, rope_mag=1.0,
                          scale=att[0].scale, freq=addr(freq))
    x = [torch.zeros(n, h * hd, device=dev) for h in (H, KH, KH)]
    seq = ints([0, 1, -1, 3], dev)
    qo = [torch.zeros(layers, n, H, hd, device=dev) for _ in range(3)]
    out = [torch.zeros(layers, n, H, hd, device=dev) for _ in range(3)]

    def step(i, st):
        p = pools[i]
        lib.pages_append(p.c, addr(seq), None, n, st)
        for l in range(layers):
            lib.qk_rope_paged_dev(p.c, heads, l, *(addr(t) for t in x), addr(seq), None, n, addr(qo[i][l]), st)
            lib.attn_paged_dev(p.c, heads, l, addr(qo[i][l]), None, addr(seq), None, n, 0, addr(out[i][l]),
                               addr(att[i].work), att[i].work.numel(), st)

    step(2, None)   # the kernels are loaded before the capture
    lib.sync()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        step(0, torch.cuda.current_stream().cuda_stream)
        err = C.c_int(0)   # reading the status of a captured stream is refused, and harms nothing
        assert lib.L.coli_hip_pages_status(C.byref(pools[0].c), None, C.byref(err),
                                           torch.cuda.current_stream().cuda_stream) == 0
    g = torch.Generator().manual_seed(2)
    for t in range(6):
        for y in x:
            y.copy_(torch.randn(y.shape, generator=g))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        step(1, None)
        lib.sync()
        assert torch.equal(out[0], out[1]) and torch.equal(qo[0], qo[1])
        for k in ("data", "table", "lens", "refs", "used"):
            assert torch.equal(getattr(pools[0], k), getattr(pools[1], k)), (t, k)
        seq.copy_(ints([0, 1, 2, -1] if t % 2 else [3, -1, 0, 2], dev))
    assert lib.pages_status(pools[0].c)[1] == 0


def test_captured_pages(mod, lib, dev):
    """Branches dropped, taken anew and grown, the pool closed up: captured once, replayed with other
    lists in the same arrays and eager work between, against the model."""
    pool = Pool(mod, lib, dev, F16, 2, 2, 32, 4, 50, 8, 10, seed=5)
    m = Model(pool)
    seq, cnt = ints([0, 1, 2, -1], dev), ints([9, 14, 4, 3], dev)
    src, dst, one = ints([0, 1, 0], dev), ints([3, 4, 5], dev), ints([1, 0, 2], dev)

    def lists(*pairs):
        for t, v in pairs:
            t.copy_(ints(v, dev))
        torch.cuda.synchronize()

    torch.cuda.synchronize()
    lib.pages_append(pool.c, addr(seq), addr(cnt), 4)
    m.append([0, 1, 2, -1], [9, 14, 4, 3])
    m.check(pool, lib, "start")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        st = torch.cuda.current_stream().cuda_stream
        lib.pages_free(pool.c, addr(dst), 3, st)
        lib.pages_fork(pool.c, addr(src), addr(dst), 3, True, st)
        lib.pages_append(pool.c, addr(dst), addr(one), 3, st)
        lib.pages_compact(pool.c, st)
    for a, b, c in (([0, 1, 0], [3, 4, 5], [1, 0, 2]), ([2, -1, 1], [5, 6, 3], [4, 1, 1]), ([1, 1, 1], [3, 4, 6], [2, 2, 2]),
                    ([0, 2, 3], [5, 6, -1], [3, 0, 9]), ([5, 0, 0], [4, 3, 7], [1, 1, 1])):
        lists((src, a), (dst, b), (one, c))
        m.free(b)
        m.fork(a, b, True)
        m.append(b, c)
        m.compact()
        graph.replay()
        torch.cuda.synchronize()
        m.check(pool, lib, (a, b, c))
        m.free([2])
        lib.pages_free(pool.c, addr(x := ints([2], dev)), 1)   # eager work between
        m.append([2], [6])
        lib.pages_append(pool.c, addr(x2 := ints([2], dev)), addr(y := ints([6], dev)), 1)
        m.check(pool, lib, "between")


# ---------------------------------------------------------------- the layer block
@pytest.mark.parametrize("dtype,n", [(F32, 1), (F32, 3), (F32, 6), (BF16, 5)], ids=lambda v: str(v))
def test_gqa_paged_block(mod, lib, orc, gen, dev, dtype, n):
    """coli_hip_gqa_paged of n sequences, tokens in step, against the CPU oracle's block per
    sequence (its dense cache): 1e-3 of the outputs as for the dense block; 16-bit pages add the
    rounding of keys and values (2^-8 of a value, 2^-8 sum |q k| of a score)."""
    _layers.bind(orc)
    D, H, KH, hd, rot, gs, max_t, layers = 256, 4, 2, 64, 16, 128, 24, 2
    W = _layers.GqaWeights(gen, gen.stream(0x9C00, n), D, H, KH, hd, rot, gs)
    tq, tk, tv, to = (m.upload(lib) for m in (W.q, W.k, W.v, W.o))
    pool = Pool(mod, lib, dev, dtype, layers, KH, hd, 4, 8 * n + 2, n + 1, 8, seed=1)
    freq = torch.tensor([float(np.float32(float(W.theta) ** (-2.0 * j / rot))) for j in range(rot // 2)], device=dev)
    qn, kn = torch.from_numpy(W.qn).to(dev), torch.from_numpy(W.kn).to(dev)
    heads = mod.Lib.heads(H=H, rot=rot, interleaved=0, q_row=2 * H * hd, q_head=2 * hd, kv_row=KH * hd, eps=1e-6,
                          rope_mag=1.0, scale=1.0 / math.sqrt(hd), qn=addr(qn), kn=addr(kn), freq=addr(freq))
    caches = [W.new_cache(max_t) for _ in range(n)]
    seq = ints(list(range(n)) + [-1], dev)
    out = torch.full((n + 1, D), 9.0, device=dev)
    for t in range(11):
        xs = np.concatenate([gen.normal(D, 0x9C10 + 100 * t + s) for s in range(n + 1)])
        x = torch.from_numpy(xs).to(dev)
        torch.cuda.synchronize()
        lib.pages_append(pool.c, addr(seq), None, n + 1)
        lib.gqa_paged_dev(pool.c, heads, 1, addr(x), tq, tk, tv, to, addr(seq), None, n + 1, t + 1, addr(out))
        sync(lib)
        got = out.cpu().numpy()
        assert not got[n].any()
        for s in range(n):
            ref = W.oracle(orc, caches[s], max_t, t, xs[s * D:(s + 1) * D])
            err = _util.maxrel_scaled(got[s], ref)
            if dtype == F32:
                assert err <= 1e-3, (t, s, err)
            else:
                e = float(np.linalg.norm(got[s] - ref) / np.linalg.norm(ref))
                # values 2^-9 in the mean, weights e^(2^-9 sqrt(sum (q k)^2)) - 1: a few 2^-9
                assert e <= 4 * 2.0 ** -8, (t, s, e)
    assert lib.pages_status(pool.c)[1] == 0


def test_gqa_paged_matches_dense(mod, lib, gen, dev):
    """A prompt in one call (rows of one sequence at their positions), against the dense block's
    token by token: the same layer over the two caches, fp32."""
    D, H, KH, hd, rot, gs, max_t, layer, S = 256, 4, 2, 64, 16, 128, 64, 150, 37
    W = _layers.GqaWeights(gen, gen.stream(0x9D00, 1), D, H, KH, hd, rot, gs)
    tq, tk, tv, to = (m.upload(lib) for m in (W.q, W.k, W.v, W.o))
    lib.kv_ensure(layer, KH * max_t, hd, hd)
    lib.gqa_norm_weight(layer, W.qn, W.kn)
    xs = np.concatenate([gen.normal(D, 0x9D10 + t) for t in range(S)])
    ref = lib.gqa_full(layer, xs, tq, tk, tv, to, S, H, KH, hd, rot, 0, max_t, W.eps, W.theta).reshape(S, D)
    pool = Pool(mod, lib, dev, F32, 1, KH, hd, 16, 5, 2, 4, seed=1)
    freq = torch.tensor([float(np.float32(float(W.theta) ** (-2.0 * j / rot))) for j in range(rot // 2)], device=dev)
    qn, kn = torch.from_numpy(W.qn).to(dev), torch.from_numpy(W.kn).to(dev)
    heads = mod.Lib.heads(H=H, rot=rot, interleaved=0, q_row=2 * H * hd, q_head=2 * hd, kv_row=KH * hd, eps=1e-6,
                          rope_mag=1.0, scale=1.0 / math.sqrt(hd), qn=addr(qn), kn=addr(kn), freq=addr(freq))
    x, out = torch.from_numpy(xs).to(dev), torch.zeros(S, D, device=dev)
    one, cnt, seq, pos = ints([1], dev), ints([S], dev), ints([1] * S, dev), ints(range(S), dev)
    torch.cuda.synchronize()
    lib.pages_append(pool.c, addr(one), addr(cnt), 1)
    lib.gqa_paged_dev(pool.c, heads, 0, addr(x), tq, tk, tv, to, addr(seq), addr(pos), S, S, addr(out))
    sync(lib)
    assert _util.maxrel_scaled(out.cpu().numpy(), ref) <= 1e-3
    for h in range(KH):
        Kd, Vd = lib.kv_read(layer, h * max_t, S, hd, hd)
        Kp, Vp = pool.rows(0, 1, S, 0)[h].numpy(), pool.rows(0, 1, S, 1)[h].numpy()
        assert np.max(np.abs(Kd - Kp)) <= 1e-4 * np.max(np.abs(Kd)) and np.max(np.abs(Vd - Vp)) <= 1e-5 * np.max(np.abs(Vd))
    side = torch.cuda.Stream()   # on a caller's stream, padded: the same rows
    again, more = torch.full((S, D), 3.0, device=dev), ints([1] * (S - 1) + [-1], dev)
    torch.cuda.synchronize()
    lib.gqa_paged_dev(pool.c, heads, 0, addr(x), tq, tk, tv, to, addr(more), addr(pos), S, 0, addr(again),
                      side.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(again[:S - 1], out[:S - 1]) and not bool(again[S - 1].any())
    L, P, h = lib.L, C.byref(pool.c), C.byref(heads)
    graph = torch.cuda.CUDAGraph()   # refused while captured, with nothing broken
    with torch.cuda.graph(graph, stream=side):
        again.zero_()
        assert L.coli_hip_gqa_paged(P, h, 0, addr(x), D, tq.handle, tk.handle, tv.handle, to.handle, addr(seq),
                                    addr(pos), S, S, addr(out), torch.cuda.current_stream().cuda_stream) == 0
    assert lib.available()
    ok = [P, h, 0, addr(x), D, tq.handle, tk.handle, tv.handle, to.handle, addr(seq), addr(pos), S, S, addr(out), None]
    for i, v in ((0, None), (1, None), (2, 1), (3, None), (4, D + 1), (5, tk.handle), (6, None), (7, tq.handle),
                 (9, None), (11, -1), (13, None)):
        args = list(ok)
        args[i] = v
        assert L.coli_hip_gqa_paged(*args) == 0, i


def test_gqa_paged_rows_past_the_end(mod, lib, gen, dev):
    """A row whose position is not held has no query: the block gives 0 for it, whatever an earlier
    call left in its scratch, and the other rows are as without it."""
    D, H, KH, hd, rot, gs = 256, 4, 2, 64, 16, 128
    W = _layers.GqaWeights(gen, gen.stream(0x9E00, 1), D, H, KH, hd, rot, gs)
    tq, tk, tv, to = (m.upload(lib) for m in (W.q, W.k, W.v, W.o))
    pool = Pool(mod, lib, dev, BF16, 1, KH, hd, 4, 12, 3, 4, seed=2)
    freq = torch.tensor([float(np.float32(float(W.theta) ** (-2.0 * j / rot))) for j in range(rot // 2)], device=dev)
    heads = mod.Lib.heads(H=H, rot=rot, interleaved=0, q_row=2 * H * hd, q_head=2 * hd, kv_row=KH * hd, eps=1e-6,
                          rope_mag=1.0, scale=1.0 / math.sqrt(hd), freq=addr(freq))
    x = torch.from_numpy(np.concatenate([gen.normal(D, 0x9E10 + t) for t in range(4)])).to(dev)

    def go(pos):
        s, p, out = ints([0, 1, 0, 2], dev), ints(pos, dev), torch.full((4, D), 4.0, device=dev)
        torch.cuda.synchronize()
        lib.gqa_paged_dev(pool.c, heads, 0, addr(x), tq, tk, tv, to, addr(s), addr(p), 4, 6, addr(out))
        sync(lib)
        return out, lib.pages_status(pool.c)[1]

    lens, cnt = ints([0, 1], dev), ints([5, 6], dev)
    torch.cuda.synchronize()
    lib.pages_append(pool.c, addr(lens), addr(cnt), 2)
    for t in range(5):   # every position written; the scratch holds queries of all rows
        go([t, t, t, -1])
    go([4, 5, 3, -1])
    whole, err = go([4, 5, 4, -1])
    assert err == 0 and bool(whole[:3].any(1).all()) and not bool(whole[3].any())
    for pos, bit in (([4, 5, 5, -1], 16), ([4, 5, 2 ** 31 - 1, 0], 16), ([4, 5, -2, -1], 4)):
        out, err = go(pos)
        assert err == bit and not bool(out[2:].any()), pos
        assert torch.equal(out[1], whole[1]), pos


@pytest.mark.parametrize("hint", [8, 40])   # a block of one wave, and of four, has a row
def test_captured_whole_rows(mod, lib, dev, hint):
    """Two captured steps with a hint, over one workspace, replayed while the sequences grow past
    the hint and rows come and go: every replay against the same call run eagerly."""
    H, KH, hd, n = 8, 2, 64, 4
    pool = Pool(mod, lib, dev, F16, 1, KH, hd, 4, 120, n, 30, seed=5)
    att = Attn(mod, lib, dev, pool, H, True, seed=6)
    lens, seq = ints([3, 0, 9, 30], dev), ints([0, 1, -1, 3], dev)
    every, more = ints(range(n), dev), ints([7, 0, 9, 11], dev)
    torch.cuda.synchronize()
    lib.pages_append(pool.c, addr(every), addr(lens), n)
    lib.sync()
    q, raw = (t.to(dev) for t in att.rows(n))
    out = [torch.full((n, H, hd), 5.0, device=dev) for _ in range(3)]

    def step(o, st):
        lib.attn_paged_dev(pool.c, att.heads, 0, addr(q), addr(raw) + 4 * hd, addr(seq), None, n, hint, addr(o),
                           addr(att.work), att.work.numel(), st)

    step(out[2], None)
    lib.sync()
    side = torch.cuda.Stream()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for i, graph in enumerate(graphs):
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            step(out[i], torch.cuda.current_stream().cuda_stream)
    for t in range(5):
        for o in out:
            o.fill_(5.0)
        torch.cuda.synchronize()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        step(out[2], None)
        lib.sync()
        assert torch.equal(out[0], out[2]) and torch.equal(out[1], out[2]), t
        att.check(torch.where(out[2] == 5.0, 77.0, out[2]).cpu(), q.cpu(), raw.cpu(), seq.tolist(),
                  [int(pool.lens[s]) if s >= 0 else 0 for s in seq.tolist()])
        lib.pages_append(pool.c, addr(every), addr(more), n)
        lib.sync()
        seq.copy_(ints([0, 1, 2, 3] if t % 2 else [3, -1, 0, 2], dev))
    assert lib.pages_status(pool.c)[1] == 0
