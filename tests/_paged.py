"""Pools of key-value pages for the tests: the device arrays of a pool, a model of its
bookkeeping in plain Python, and 64-bit forms of the operators over it (CPU)."""
import math

import numpy as np
import torch

F32, F16, BF16 = 0, 1, 2
TORCH = {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}
NAMES = {F32: "f32", F16: "f16", BF16: "bf16"}
U = 2.0 ** -24   # half a step of fp32, relative


def ints(v, dev):
    return torch.tensor(list(v), dtype=torch.int32, device=dev)


def addr(t):
    return None if t is None else t.data_ptr()


class Pool:
    """The arrays of a pool on `dev` and its ColiHipPages.  data starts as random values."""

    def __init__(self, mod, lib, dev, dtype, layers, KH, hd, page, n_pages, n_seqs, max_pages, seed=0, init=True,
                 fill=True):
        g = torch.Generator().manual_seed(seed)
        shape = (n_pages, layers, 2, KH, page, hd)
        self.dtype, self.layers, self.KH, self.hd, self.page = dtype, layers, KH, hd, page
        self.n_pages, self.n_seqs, self.max_pages, self.dev = n_pages, n_seqs, max_pages, dev
        if fill:
            self.data = torch.randn(shape, generator=g).to(TORCH[dtype]).to(dev)
        else:
            self.data = torch.zeros(shape, dtype=TORCH[dtype], device=dev)
        i32 = dict(dtype=torch.int32, device=dev)
        self.table, self.lens = torch.full((n_seqs, max_pages), 77, **i32), torch.full((n_seqs,), 5, **i32)
        self.refs, self.used = torch.full((n_pages,), 3, **i32), torch.full(((n_pages + 31) // 32,), 9, **i32)
        self.state = torch.full((mod.Lib.PAGES_STATE,), 1, **i32)
        self.work = torch.full((lib.pages_work(n_seqs, n_pages),), -7, **i32)
        self.c = mod.Lib.pages(*(addr(t) for t in (self.data, self.table, self.lens, self.refs, self.used, self.state,
                                                   self.work)), dtype, layers, KH, hd, page, n_pages, n_seqs, max_pages)
        if init:
            torch.cuda.synchronize()
            lib.pages_init(self.c)
            lib.sync()

    def place(self, lens, seed=1):
        """Sequences 0.. of the given lengths on scattered pages, written to the arrays."""
        rng = np.random.default_rng(seed)
        ids = rng.permutation(self.n_pages)
        table, refs, at = np.full((self.n_seqs, self.max_pages), -1, np.int32), np.zeros(self.n_pages, np.int32), 0
        for s, x in enumerate(lens):
            k = -(-x // self.page)
            table[s, :k] = ids[at:at + k]
            refs[ids[at:at + k]] = 1
            at += k
        self.table.copy_(torch.from_numpy(table))
        self.refs.copy_(torch.from_numpy(refs))
        self.lens.copy_(torch.tensor(list(lens) + [0] * (self.n_seqs - len(lens)), dtype=torch.int32))
        self.used.copy_(torch.from_numpy(bitmap(refs)))
        self.state.zero_()
        torch.cuda.synchronize()

    def rows(self, layer, s, n, kv):
        """K (kv 0) or V rows 0..n-1 of sequence s in 64 bits [KH, n, hd], from the arrays."""
        pg = self.table[s, :-(-n // self.page)].long().to(self.data.device)
        x = self.data[pg, layer, kv].cpu()           # [P, KH, page, hd]
        return x.permute(1, 0, 2, 3).reshape(self.KH, -1, self.hd)[:, :n].double()


def bitmap(refs):
    n = len(refs)
    bits = np.zeros(-(-n // 32) * 32, np.uint8)
    bits[:n] = np.asarray(refs) > 0
    return np.packbits(bits.reshape(-1, 8), axis=1, bitorder="little").reshape(-1).view(np.uint32).view(np.int32).copy()


class Model:
    """What the pool's bookkeeping has to come to: plain lists, pages as (sequence of rows)."""

    def __init__(self, pool):
        self.page, self.n_pages, self.max_pages = pool.page, pool.n_pages, pool.max_pages
        self.pages = [[] for _ in range(pool.n_seqs)]
        self.lens, self.refs = [0] * pool.n_seqs, [0] * pool.n_pages
        self.data = pool.data.cpu().clone()
        self.err = 0

    def _take(self, k):
        free = [p for p in range(self.n_pages) if not self.refs[p]]
        return None if k > len(free) else free[:k]

    def _bad(self, bit):
        self.err |= bit
        return False

    def append(self, seqs, counts=None):
        counts = [1] * len(seqs) if counts is None else list(counts)
        live = [(s, c) for s, c in zip(seqs, counts) if s != -1]
        bad = 0
        if any(s < -1 or s >= len(self.lens) for s, _ in live) or any(c < 0 for _, c in live):
            bad |= 4
        good = [(s, c) for s, c in live if 0 <= s < len(self.lens) and c >= 0]
        if len({s for s, _ in good}) < len(good):
            bad |= 8
        if any(self.lens[s] + c > self.max_pages * self.page for s, c in good):
            bad |= 2
        if bad:
            return self._bad(bad)
        need = [-(-(self.lens[s] + c) // self.page) - len(self.pages[s]) for s, c in live]
        new = self._take(sum(need))
        if new is None:
            return self._bad(1)
        for (s, c), k in zip(live, need):
            for p in new[:k]:
                self.pages[s].append(p)
                self.refs[p] = 1
            new = new[k:]
            self.lens[s] += c
        return True

    def fork(self, src, dst, share):
        pairs = [(a, b) for a, b in zip(src, dst) if a != -1 and b != -1]
        n = len(self.lens)
        if any(not (-1 <= x < n) for x in list(src) + list(dst)):
            return self._bad(4)
        if any(a == b or self.lens[b] for a, b in pairs) or len({b for _, b in pairs}) < len(pairs):
            return self._bad(8)
        old = {a: (list(self.pages[a]), self.lens[a]) for a, _ in pairs}
        need = [int(old[a][1] % self.page != 0) if share else len(old[a][0]) for a, _ in pairs]
        new = self._take(sum(need))
        if new is None:
            return self._bad(1)
        for (a, b), k in zip(pairs, need):
            got, new = new[:k], new[k:]
            pages, length = old[a]
            keep = length // self.page if share else 0
            for p in pages[:keep]:
                self.refs[p] += 1
            for j, p in enumerate(got):
                held = min(self.page, length - (keep + j) * self.page)
                self.data[p, ..., :held, :] = self.data[pages[keep + j], ..., :held, :]
                self.refs[p] = 1
            self.pages[b], self.lens[b] = pages[:keep] + got, length
        return True

    def free(self, seqs):
        for s in seqs:
            if s == -1:
                continue
            if not 0 <= s < len(self.lens):
                self.err |= 4
                continue
            for p in self.pages[s]:
                self.refs[p] -= 1
            self.pages[s], self.lens[s] = [], 0

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        holes = [p for p in range(live) if not self.refs[p]]
        movers = [p for p in range(live, self.n_pages) if self.refs[p]]
        to = dict(zip(movers, holes))
        for m, h in to.items():
            self.data[h] = self.data[m]
            self.refs[h], self.refs[m] = self.refs[m], 0
        self.pages = [[to.get(p, p) for p in row] for row in self.pages]

    def check(self, pool, lib, what):
        free, err = lib.pages_status(pool.c)
        assert err == self.err, (what, err, self.err)
        self.err = 0
        table = np.full((len(self.lens), self.max_pages), -1, np.int32)
        for s, row in enumerate(self.pages):
            table[s, :len(row)] = row
        assert pool.lens.tolist() == self.lens, what
        assert np.array_equal(pool.table.cpu().numpy(), table), what
        assert pool.refs.tolist() == self.refs, what
        assert np.array_equal(pool.used.cpu().numpy(), bitmap(self.refs)), what
        assert free == sum(r == 0 for r in self.refs), what
        got = pool.data.cpu()
        assert torch.equal(got.view(torch.int16 if got.element_size() == 2 else torch.int32),
                           self.data.view(torch.int16 if got.element_size() == 2 else torch.int32)), what


# ---------------------------------------------------------------- the operators in 64 bits
def norm64(x, w, eps):
    x = x.double()
    if w is None:
        return x
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * (1.0 + w.double())


def rope64(x, pos, freq, rot, interleaved, mag):
    """x [n, heads, hd], pos [n] -> (rotated, |u| + |v| of each output's pair)."""
    y, size = x.clone(), x.abs()
    if rot:
        a = pos.double()[:, None] * freq.double()
        c, s = (torch.cos(a) * mag)[:, None], (torch.sin(a) * mag)[:, None]
        i = torch.arange(rot // 2)
        fst, snd = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
        u, v = x[..., fst], x[..., snd]
        y[..., fst], y[..., snd] = u * c - v * s, v * c + u * s
        size[..., fst] = size[..., snd] = (u.abs() + v.abs()) * max(1.0, abs(mag))
    return y, size


def attn(q, K, V, scale, gate=None, dtype=torch.float64):
    """q [H, hd] over K, V [KH, n, hd]: (out [H, hd], sum p |v|, largest scale sum |q k|)."""
    H, (KH, n, hd) = q.shape[0], K.shape
    q, K, V = q.to(dtype), K.to(dtype), V.to(dtype)
    if n == 0:
        z = torch.zeros(H, hd, dtype=dtype)
        return z, z, 0.0
    qg = q.view(KH, H // KH, hd)
    s = qg @ K.transpose(1, 2) * scale
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o, size = (p @ V).reshape(H, hd), (p @ V.abs()).reshape(H, hd)
    big = float((qg.abs() @ K.abs().transpose(1, 2)).max()) * abs(scale)
    if gate is not None:
        g = 1.0 / (1.0 + torch.exp(-gate.to(dtype)))
        o, size = o * g, size * g
    return o, size, big


def attn_bound(size, big, hd, n):
    """Elementwise bound of an fp32 evaluation against 64 bits.  A dot of hd terms is off by at
    most lambda sqrt(hd) U times its absolute sum but with negligible probability (lambda = 6,
    independent roundings); a score error e changes a softmax's outputs by at most 2 e sum p |v|;
    exponentials, weights, the sums over n keys (lambda sqrt(n)), the division and the gate's
    sigmoid (scores and differences of up to `big`, rounded once more each) add the rest."""
    return U * (2 * (6 * math.sqrt(hd) * big + 4 * big + 4) + 6 * math.sqrt(max(n, 1)) + 24) * size + 1e-37
