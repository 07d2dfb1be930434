"""The several-sequences operators without a GPU: how the attention kernels divide their work (every unit of every item exactly
once, whatever the lengths), and the refusals of the entry points and of the Python layer, which come before any launch."""
import ctypes as C

import numpy as np
import pytest

from jitllm_b200 import _lib

L = _lib.load()


def _shares(starts, lens, total, hkv, tok_item, shift, min_units, page_shift, max_pages, grid):
    starts = np.asarray(starts, np.int32)
    lens = None if lens is None else np.asarray(lens, np.int32)
    out = []
    segs = np.zeros((1 << 16, 6), np.int32)
    for c in range(grid):
        n = L.jl_test_attn_share(starts.ctypes.data, lens.ctypes.data if lens is not None else None, len(starts) - 1, total, hkv, tok_item,
                                 shift, min_units, page_shift, max_pages, grid, c, segs.ctypes.data, len(segs))
        assert n >= 0
        out.append(segs[:n].tolist())
    return out


def _items(starts, lens, total, hkv, T, shift, page_shift, max_pages):
    items = {}
    for s in range(len(starts) - 1):
        lo = min(max(starts[s], 0), total)
        n = min(max(starts[s + 1], lo), total) - lo
        ln = max(0, lens[s]) if lens is not None else n
        pos0 = ln - n
        if max_pages:
            ln = min(ln, max_pages << page_shift)
        for b in range(-(-n // T)):
            limit = min(max(pos0 + min((b + 1) * T, n), 0), ln)
            for h in range(hkv):
                items[(s, b, h)] = -(-limit // (1 << shift))
    return items


CASES = [
    dict(new=[1], lens=[2049], hkv=8, T=4, shift=6, grid=444),
    dict(new=[1] * 40, lens=list(range(1, 8001, 200)), hkv=8, T=4, shift=6, grid=444),
    dict(new=[0, 5, 0, 0, 300, 1, 0], lens=[7, 5, 0, 90, 1000, 0, 33], hkv=2, T=5, shift=6, grid=37),    # idle ones, an empty one
    dict(new=[1531], lens=None, hkv=8, T=64, shift=7, grid=148),
    dict(new=[1, 2, 3, 129, 64, 700, 0, 8], lens=None, hkv=3, T=42, shift=7, grid=148),
    dict(new=[16384], lens=None, hkv=1, T=64, shift=7, grid=148),
    dict(new=[9, 9], lens=[3, 200], hkv=2, T=4, shift=6, grid=11),                                       # shorter than its new rows
    dict(new=[1], lens=[131071], hkv=2, T=2, shift=6, grid=444),
    dict(new=[2, 2], lens=[5000, 100], hkv=2, T=2, shift=6, grid=20, max_pages=4),                       # longer than its table
    dict(new=[1] * 70, lens=[0] * 70, hkv=2, T=4, shift=6, grid=12),                                     # nothing to read at all
]


@pytest.mark.parametrize("c", CASES)
@pytest.mark.parametrize("min_units", [1, 2, 7])
def test_every_unit_is_somebodys(c, min_units):
    starts = [0]
    for n in c["new"]:
        starts.append(starts[-1] + n)
    total, mp = starts[-1] + 3, c.get("max_pages", 0)
    shares = _shares(starts, c["lens"], total, c["hkv"], c["T"], c["shift"], min_units, 6, mp, c["grid"])
    items = _items(starts, c["lens"], total, c["hkv"], c["T"], c["shift"], 6, mp)
    seen, order = {k: [] for k in items}, []
    for cta, segs in enumerate(shares):
        for i, (s, b, h, u0, u1, units) in enumerate(segs):
            assert units == items[(s, b, h)]
            assert 0 <= u0 <= u1 <= units and (u0 < u1 or units == 0)
            if u0 > 0:
                assert i == 0                                    # only a share's first segment continues an item
            if u1 < units:
                assert i == len(segs) - 1                        # only its last one leaves an item open
            seen[(s, b, h)].append((u0, u1))
            order.append((s, b, h, u0))
    assert order == sorted(order)
    for k, parts in seen.items():
        at = 0
        if items[k] == 0:
            assert parts == [(0, 0)]
            continue
        for u0, u1 in parts:
            assert u0 == at
            at = u1
        assert at == items[k]


def test_shares_are_even():
    """Long items: no CTA takes much more than the mean."""
    starts, lens = [0, 1, 2, 3], [131072, 70000, 12]
    shares = _shares(starts, lens, 3, 8, 4, 6, 2, 6, 0, 444)
    work = [sum(u1 - u0 for _, _, _, u0, u1, _ in segs) for segs in shares]
    assert max(work) <= 1.15 * sum(work) / len(work) + 2


def test_random_sequences():
    rng = np.random.default_rng(5)
    for _ in range(60):
        n = int(rng.integers(1, 50))
        new = rng.integers(0, 40, n).tolist()
        lens = [int(x + rng.integers(-5, 900)) for x in new]
        starts = np.concatenate([[0], np.cumsum(new)]).tolist()
        if starts[-1] == 0:
            continue
        hkv, T, grid = int(rng.integers(1, 9)), int(rng.integers(1, 17)), int(rng.integers(1, 300))
        items = _items(starts, lens, starts[-1], hkv, T, 6, 4, 9)
        got = {}
        for segs in _shares(starts, lens, starts[-1], hkv, T, 6, int(rng.integers(1, 5)), 4, 9, grid):
            for s, b, h, u0, u1, _ in segs:
                got[(s, b, h)] = got.get((s, b, h), 0) + (u1 - u0 if items[(s, b, h)] else 1)
        assert got == {k: max(v, 1) for k, v in items.items()}


def test_hostile_starts_stay_inside_the_rows():
    """starts that fall, are negative or pass the rows: the segments stay within [0, total)."""
    for starts in ([5, 2, 9, -4, 3], [-7, 100, 4], [0, 1 << 30]):
        for segs in _shares(starts, None, 12, 2, 4, 6, 1, 6, 0, 9):
            for s, b, h, u0, u1, units in segs:
                lo = min(max(starts[s], 0), 12)
                assert lo + b * 4 < 12


def test_entry_points_refuse_without_a_context():
    kv = _lib.PagedKVDesc(struct_size=C.sizeof(_lib.PagedKVDesc))
    assert C.sizeof(_lib.PagedKVDesc) == 56
    assert L.jl_attn_scratch_bytes(None) == 0
    assert L.jl_attn_prompt(None, 16, 0, 16, 128, 128, 16, 16, 128, 128, 2, 16, 1, 1, 1, 1, 128, 1.0, 16, 1 << 30, None) == _lib.EINVAL
    assert L.jl_attn_paged(None, 16, 0, 16, 128, 128, C.byref(kv), 16, 16, 1, 1, 1, 1.0, 16, 1 << 30, None) == _lib.EINVAL
    assert L.jl_rope_append(None, 16, 16, 0, C.byref(kv), 16, 16, 1, 1, 16, 16, 1, None) == _lib.EINVAL
    s = np.zeros(2, np.int32)
    assert L.jl_test_attn_share(s.ctypes.data, None, 0, 1, 1, 1, 6, 1, 6, 0, 1, 0, s.ctypes.data, 0) == _lib.EINVAL


@pytest.mark.parametrize("length", [2 ** 31 - 1, 2 ** 31 - 257, 2 ** 30 + 1, 5000])
def test_a_length_beyond_its_table_takes_no_more_than_the_table(length):
    """One sequence claims more positions than its table holds: it weighs what the table holds, and the others get their shares of the
    grid. (The claimed length would take all of it; near 2^31 its sum with an item's cost left 32 bits.)"""
    starts, lens = [0, 1, 2, 3], [1280, length, 1280]                    # tables of 20 pages of 64
    shares = _shares(starts, lens, 3, 8, 4, 6, 2, 6, 20, 100)
    work = [sum(u1 - u0 for _, _, _, u0, u1, _ in segs) for segs in shares]
    assert sum(work) == 3 * 8 * 20 and max(work) <= 1.15 * sum(work) / len(work) + 2
    for s in (0, 1, 2):
        assert len([c for c, segs in enumerate(shares) if any(g[0] == s for g in segs)]) >= 20


@pytest.mark.parametrize("name", ["attn.cu", "attn.cuh", "attn_few.cu", "attn_tc5.cu"])
def test_no_read_only_loads_behind_a_dependent_launch(name):
    """These kernels are put in place while the one in front of them still runs, and what they read that one may have written: the read-only
    load is for memory that nothing writes while a kernel is there."""
    import os
    from jitllm_b200 import build
    text = open(os.path.join(build.CSRC, name)).read()
    assert "__ldg(" not in text and "global.nc" not in text and "__restrict__" not in text


@pytest.mark.parametrize("dtype", ["uint32", "int64", "int16", "float32"])
def test_a_page_table_is_int32(dtype):
    import torch
    from jitllm_b200 import PagedKV
    k = torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="int32"):
        PagedKV(k, k.clone(), torch.zeros(1, 2, dtype=getattr(torch, dtype)))


# what the kernels are launched with: unit, an item's cost, snap, tokens of an item, CTAs
LAUNCHED = {"few": (6, 4, 2, lambda g: 16 // g, 444), "two tiles": (7, 3, 1, lambda g: 2 * (128 // g), 148), "one tile": (7, 2, 0, lambda g: 128 // g, 296)}
TAKES = {"all": (0, 2 ** 31 - 1), "up to sixteen rows": (0, 16), "more": (16, 2 ** 31 - 1)}


@pytest.mark.parametrize("which", LAUNCHED)
@pytest.mark.parametrize("takes", TAKES)
def test_the_launches_own_divisions(which, takes):
    """Lengths, groups and idle sequences at random: of the sequences that a launch takes every unit of every item falls to one CTA, and the
    parts of an item that a join would follow from the CTA that began it are all of them, in ascending order."""
    shift, cost, snap, tokens, grid = LAUNCHED[which]
    lo, hi = TAKES[takes]
    rng = np.random.default_rng(11)
    segs = np.zeros((1 << 14, 6), np.int32)
    for trial in range(25):
        n, g, hkv = int(rng.integers(1, 200)), int(rng.choice([1, 2, 3, 4, 8, 16])), int(rng.integers(1, 9))
        new = np.where(rng.random(n) < 0.3, 0, np.where(rng.random(n) < 0.6, 1, rng.integers(1, 200, n)))
        lens = np.maximum(0, new + rng.integers(-3, rng.choice([40, 3000, 9000]), n)).astype(np.int32)
        starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        if trial % 5 == 0:
            lens[rng.integers(0, n)] = 2 ** 31 - 1
        total, T, max_pages = int(starts[-1]), tokens(g), 130
        if total == 0:
            continue
        items = {}
        for s in range(n):
            if not lo < new[s] * g <= hi:
                continue
            pos0, ln = int(lens[s]) - int(new[s]), min(int(lens[s]), max_pages << 6)
            for b in range(-(-int(new[s]) // T)):
                limit = min(max(pos0 + min((b + 1) * T, int(new[s])), 0), ln)
                for h in range(hkv):
                    items[(s, b, h)] = -(-limit // (1 << shift))
        shares = []
        for c in range(grid):
            k = L.jl_test_attn_share_as(starts.ctypes.data, lens.ctypes.data, n, total, hkv, g, lo, hi, T, cost, snap, shift, 2, 6, max_pages, grid,
                                        c, segs.ctypes.data, len(segs))
            assert k >= 0
            shares.append(segs[:k].tolist())
        whole, own, cont = [], {}, {}
        for c, share in enumerate(shares):
            for i, (s, b, h, u0, u1, units) in enumerate(share):
                assert units == items[(s, b, h)] and (0 <= u0 < u1 <= units or u0 == u1 == units == 0)
                if u0 == 0 and u1 == units:
                    whole.append((s, b, h))
                elif u0 > 0:
                    assert i == 0 and c not in cont              # slot 0
                    cont[c] = ((s, b, h), u0, u1, u1 == units)
                else:
                    assert i == len(share) - 1 and c not in own  # slot 1
                    own[c] = ((s, b, h), u1)
        for c, (item, at) in own.items():                        # as the join goes on from there
            d = c + 1
            while True:
                assert d < grid
                if d in cont:
                    assert cont[d][0] == item and cont[d][1] == at
                    at = cont[d][2]
                    if cont.pop(d)[3]:
                        break
                else:
                    assert not shares[d]
                d += 1
            assert at == items[item]
            whole.append(item)
        assert not cont and sorted(whole) == sorted(items)


def test_shares_of_nothing_are_refused():
    """Settings that would divide by zero or shift out of range come back as an error."""
    s = np.zeros(6, np.int32)
    good = dict(nseq=1, total=1, hkv=1, g=1, row_lo=0, row_hi=9, tok_item=1, item_cost=1, snap=0, unit_shift=6, min_units=1, page_shift=6, max_pages=0, grid=1, cta=0)

    def call(**kw):
        return L.jl_test_attn_share_as(s.ctypes.data, None, *{**good, **kw}.values(), s.ctypes.data, 1)
    assert call() >= 0
    for bad in (dict(min_units=0), dict(g=0), dict(tok_item=0), dict(unit_shift=0), dict(unit_shift=40), dict(page_shift=-1), dict(page_shift=40), dict(grid=0),
                dict(cta=1), dict(cta=-1), dict(nseq=0), dict(hkv=0), dict(item_cost=-1), dict(snap=-1)):
        assert call(**bad) == _lib.EINVAL, bad
    assert L.jl_test_attn_share(s.ctypes.data, None, 1, 1, 1, 1, 6, 0, 6, 0, 1, 0, s.ctypes.data, 1) == _lib.EINVAL
