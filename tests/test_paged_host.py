"""The paged cache's checks of its arguments, on the host alone: descriptions it refuses, and
every call of a process without a device returning 0."""
import ctypes as C

import pytest
import torch

import _util


@pytest.fixture(scope="module")
def mod():
    return _util.load_product()


@pytest.fixture(scope="module")
def bare(mod):
    return mod.Lib()   # not initialised: no device


GOOD = dict(data=0x1000, table=0x2000, lens=0x3000, refs=0x4000, used=0x5000, state=0x6000, work=0x7000, dtype=2,
            n_layers=2, KH=2, hd=64, page=16, n_pages=10, n_seqs=3, max_pages=4)
HEADS = dict(H=8, rot=32, interleaved=0, q_row=1024, q_head=128, kv_row=128, eps=1e-6, rope_mag=1.0, scale=0.125,
             qn=0x1000, kn=0x1000, freq=0x1000)


def test_good_description(mod, bare):
    assert bare.L.coli_hip_pages_check(C.byref(mod.Lib.pages(**GOOD))) == 1
    assert bare.L.coli_hip_heads_check(C.byref(mod.Lib.pages(**GOOD)), C.byref(mod.Lib.heads(**HEADS))) == 1
    assert bare.pages_work(3, 10) >= 3 + 2 * 10
    assert bare.L.coli_hip_pages_work(None) == 0


@pytest.mark.parametrize("change", [
    dict(data=None), dict(table=None), dict(lens=None), dict(refs=None), dict(used=None), dict(state=None),
    dict(work=None), dict(data=0x1008), dict(dtype=3), dict(dtype=-1), dict(hd=0), dict(hd=4), dict(hd=60),
    dict(hd=264), dict(page=0), dict(page=4097), dict(KH=0), dict(n_layers=0), dict(n_pages=0), dict(n_seqs=0),
    dict(max_pages=0), dict(max_pages=1 << 28), dict(n_pages=(1 << 30) + 1),
], ids=str)
def test_refused_pools(mod, bare, change):
    assert bare.L.coli_hip_pages_check(C.byref(mod.Lib.pages(**dict(GOOD, **change)))) == 0
    assert bare.L.coli_hip_heads_check(C.byref(mod.Lib.pages(**dict(GOOD, **change))),
                                       C.byref(mod.Lib.heads(**HEADS))) == 0


@pytest.mark.parametrize("change", [
    dict(H=0), dict(H=7), dict(H=-2), dict(rot=31), dict(rot=66), dict(rot=-2), dict(freq=None), dict(q_head=63),
    dict(q_row=7 * 128 + 63), dict(kv_row=127),
], ids=str)
def test_refused_heads(mod, bare, change):
    p = mod.Lib.pages(**GOOD)
    assert bare.L.coli_hip_heads_check(C.byref(p), C.byref(mod.Lib.heads(**dict(HEADS, **change)))) == 0
    assert bare.L.coli_hip_attn_paged_work(C.byref(p), C.byref(mod.Lib.heads(**dict(HEADS, **change)))) == 0


def test_accepted_heads(mod, bare):
    """No rotation needs no frequencies; no norms; one head; rows side by side."""
    p = mod.Lib.pages(**GOOD)
    for change in (dict(rot=0, freq=None), dict(qn=None, kn=None), dict(H=2, q_row=128, q_head=64), dict(rot=64)):
        h = mod.Lib.heads(**dict(HEADS, **change))
        assert bare.L.coli_hip_heads_check(C.byref(p), C.byref(h)) == 1
        assert bare.L.coli_hip_attn_paged_work(C.byref(p), C.byref(h)) > 0


def test_no_device_no_work(mod, bare):
    """Without coli_vk_init every call returns 0 and touches nothing (the addresses are no memory)."""
    if torch.cuda.is_available():
        pytest.skip("a device is present")
    L, p, h = bare.L, C.byref(mod.Lib.pages(**GOOD)), C.byref(mod.Lib.heads(**HEADS))
    a = 0x1000
    assert L.coli_hip_pages_init(p, None) == 0
    assert L.coli_hip_pages_append(p, a, a, 2, None) == 0
    assert L.coli_hip_pages_fork(p, a, a, 2, 1, None) == 0
    assert L.coli_hip_pages_free(p, a, 2, None) == 0
    assert L.coli_hip_pages_compact(p, None) == 0
    assert L.coli_hip_pages_status(p, None, None, None) == 0
    assert L.coli_hip_qk_rope_paged(p, h, 0, a, a, a, a, None, 2, a, None) == 0
    assert L.coli_hip_attn_paged(p, h, 0, a, None, a, None, 2, 0, a, a, 1 << 30, None) == 0
    assert L.coli_hip_gqa_paged(p, h, 0, a, 64, None, None, None, None, a, None, 2, 0, a, None) == 0


@pytest.mark.parametrize("change", [dict(q_row=(1 << 40) + 1), dict(q_head=1 << 60, q_row=1 << 62),
                                    dict(kv_row=1 << 62)], ids=str)
def test_refused_far_strides(mod, bare, change):
    """Offsets of a call's rows stay within 64 bits."""
    p, h = mod.Lib.pages(**GOOD), mod.Lib.heads(**dict(HEADS, **change))
    assert bare.L.coli_hip_heads_check(C.byref(p), C.byref(h)) == 0
