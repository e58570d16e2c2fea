"""Rotary positions, the 8-bit token cache, attention over it and the gated norm, each through the C ABI against its definition in
64 bits (token_ops_ref.py, which also derives the bounds)."""
import math
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import token_ops_ref as R  # noqa: E402
from video_depth_anything import hip  # noqa: E402

DEV = "cuda"
HALVES = [torch.bfloat16, torch.float16]
TYPES = HALVES + [torch.float32]
PAIR = {"halves": hip.PAIR_HALVES, "adjacent": hip.PAIR_ADJACENT}
FMT = {"i8": hip.CACHE_I8, "e4m3": hip.CACHE_E4M3}
NORM = {"none": hip.NORM_NONE, "layer": hip.NORM_LAYER, "rms": hip.NORM_RMS}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def within(got, want, tol, what=""):
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    fine = ~torch.isnan(want)
    over = ((got - want).abs() - tol)[fine]
    assert over.numel() == 0 or float(over.max()) <= 0, f"{what}: {float(over.max()):.3e} beyond the bound, of {float(want[fine].abs().max()):.3e}"


# ---- rotary positions ------------------------------------------------------------------------------------------------------
def rotary_inputs(rows, heads, hd, n, dt, seed, far=False, pos_float=False):
    g = gen(seed)
    x = torch.randn((rows, heads, hd), generator=g).to(dt).to(DEV)
    pos = torch.randint(-5_000_000 if far else -40, 5_000_000 if far else 2000, (rows, 3), generator=g)
    pos = (pos.float() * 0.37 if pos_float else pos.to(torch.int32)).to(DEV)
    freq = (torch.rand(n, generator=g, dtype=torch.float64) * 2).to(DEV)
    return x, pos, freq


def rotary_check(got, x, pos, freq, sections, pairing):
    want, size = R.rotate(x, pos, freq, sections, pairing)
    d = R.ROTATION * size
    within(got, want, d + (0 if x.dtype == torch.float32 else R.half_step(x.dtype)) * (want.abs() + d) + 2.0 ** -25, pairing)


@pytest.mark.parametrize("pairing", ["halves", "adjacent"])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,heads,hd,sections", [(1, 1, 8, (4, 0, 0)), (1, 12, 64, (8, 12, 12)), (37, 6, 64, (0, 8, 8)), (1371, 3, 48, (6, 9, 9)),
                                                    (2050, 2, 24, (1, 1, 2)), (5, 32, 128, (16, 24, 24)), (66, 5, 96, (4, 20, 16)), (9, 2, 256, (40, 44, 44))])
def test_rotary_turns_every_pair(rows, heads, hd, sections, dt, pairing):
    x, pos, freq = rotary_inputs(rows, heads, hd, sum(sections), dt, rows + hd)
    out = torch.full_like(x, float("nan"))
    hip.rotary_axes(x, out, pos, freq, rows=rows, heads=heads, hd=hd, sections=sections, pairing=PAIR[pairing])
    rotary_check(out, x, pos, freq, sections, pairing)
    y = x.clone()
    hip.rotary_axes(y, y, pos, freq, rows=rows, heads=heads, hd=hd, sections=sections, pairing=PAIR[pairing])
    assert torch.equal(y, out)


@pytest.mark.parametrize("pos_float", [False, True])
@pytest.mark.parametrize("dt", TYPES)
def test_rotary_far_positions(dt, pos_float):
    """Positions of millions, whose fp32 angles are off by tenths of a radian."""
    x, pos, freq = rotary_inputs(300, 4, 64, 32, dt, 5, far=True, pos_float=pos_float)
    out = torch.empty_like(x)
    hip.rotary_axes(x, out, pos, freq, rows=300, heads=4, hd=64, sections=(10, 11, 11))
    rotary_check(out, x, pos, freq, (10, 11, 11), "halves")


@pytest.mark.parametrize("dt", TYPES)
def test_rotary_of_q_and_k_inside_packed_rows(dt):
    """q and k of a packed [q | k | v] row in one call, in place: v and the rest of the buffer stay bit for bit."""
    rows, heads, hd = 70, 3, 32
    buf = torch.randn((rows + 2, 3 * heads * hd + 16), generator=gen(3)).to(dt).to(DEV)
    was = buf.clone()
    view = buf[1:rows + 1, :2 * heads * hd]
    _, pos, freq = rotary_inputs(rows, 1, hd, 16, dt, 4)
    hip.rotary_axes(view, view, pos, freq, rows=rows, heads=2 * heads, hd=hd, sections=(4, 6, 6))
    rotary_check(view.reshape(rows, 2 * heads, hd), was[1:rows + 1, :2 * heads * hd].reshape(rows, 2 * heads, hd), pos, freq, (4, 6, 6), "halves")
    assert torch.equal(buf[:, 2 * heads * hd:], was[:, 2 * heads * hd:]) and torch.equal(buf[0], was[0]) and torch.equal(buf[-1], was[-1])


def test_rotary_with_negated_frequencies_is_the_inverse_and_the_gradient():
    """The rotation is orthogonal: turned back it is the input, and the gradient of <w, rotate(x)> with respect to x is w turned back."""
    x, pos, freq = rotary_inputs(50, 2, 64, 32, torch.float32, 8)
    y, z = torch.empty_like(x), torch.empty_like(x)
    kw = dict(rows=50, heads=2, hd=64, sections=(8, 12, 12))
    hip.rotary_axes(x, y, pos, freq, **kw)
    hip.rotary_axes(y, z, pos, -freq, **kw)
    size = R.rotate(x, pos, freq, (8, 12, 12), "halves")[1]
    within(z, x.double().cpu(), 4 * R.ROTATION * size)
    w, gx = torch.randn(x.shape, generator=gen(9)).to(DEV), torch.empty_like(x)
    hip.rotary_axes(w, gx, pos, -freq, **kw)
    a = x.double().cpu().requires_grad_(True)
    (R.rotate(a.detach(), pos, freq, (8, 12, 12), "halves")[0] * 0).sum()
    step = torch.randn(x.shape, generator=gen(10), dtype=torch.float64)
    f = lambda v: float((w.double().cpu() * R.rotate(v, pos, freq, (8, 12, 12), "halves")[0]).sum())  # noqa: E731
    base = x.double().cpu()
    difference = f(base + step) - f(base)                 # the map is linear: the difference is the derivative
    assert abs(difference - float((gx.double().cpu() * step).sum())) <= 4 * R.ROTATION * float((w.abs().cpu().double().sum() * step.abs().max()))


# ---- the cache ---------------------------------------------------------------------------------------------------------------
def new_cache(pages, kv_heads, page, hd, fill=0):
    code = lambda: torch.full((pages, kv_heads, page, hip.cache_row_bytes(hd)), fill, dtype=torch.uint8, device=DEV)  # noqa: E731
    exps = lambda: torch.zeros((pages, kv_heads, page), dtype=torch.uint8, device=DEV)  # noqa: E731
    return code(), code(), exps(), exps()


def cache_rows(rows, kv_heads, hd, dt, seed):
    """Rows of very different sizes, some of zeros, of one value, of the type's extremes, with ties between codes."""
    g = gen(seed)
    x = torch.randn((rows, kv_heads, hd), generator=g) * torch.exp2(torch.randint(-12, 13, (rows, kv_heads, 1), generator=g).float())
    x[::7] = torch.round(torch.randn(x[::7].shape, generator=g) * 20) / 2            # halves: ties between neighbouring codes
    x = x.to(dt)
    if rows > 3:
        x[1] = 0
        x[2, :, 0] = torch.finfo(dt).max
        x[3] = torch.finfo(dt).tiny
    return x.to(DEV)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,kv_heads,hd,page", [(1, 1, 8, 16), (1, 6, 64, 1376), (45, 3, 24, 16), (2100, 2, 32, 48), (100, 4, 48, 64), (33, 16, 64, 16),
                                                   (77, 2, 96, 32), (260, 1, 128, 1376), (50, 5, 16, 16), (20, 3, 40, 32)])
def test_cache_write_stores_the_rules_codes_and_reads_back(rows, kv_heads, hd, page, dt, fmt):
    pages = -(-rows // page) + 3
    slots = torch.randperm(pages * page, generator=gen(rows))[:rows].to(DEV)
    if rows > 10:
        slots[4], slots[9] = -1, pages * page + 5                               # rows without a slot
    k, v = cache_rows(rows, kv_heads, hd, dt, 1), cache_rows(rows, kv_heads, hd, dt, 2)
    ck, cv, ek, ev = new_cache(pages, kv_heads, page, hd, fill=0xAB)
    kw = dict(rows=rows, kv_heads=kv_heads, hd=hd, page_size=page, fmt=FMT[fmt])
    hip.cache_write(k, v, ck, cv, ek, ev, slots, **kw)
    here = (slots >= 0) & (slots < pages * page)
    p, o = slots[here] // page, slots[here] % page
    for x, c, e in ((k, ck, ek), (v, cv, ev)):
        want_e = R.exponents(x[here].cpu(), fmt)
        assert torch.equal(e[p, :, o].cpu().long(), want_e)
        raw = c[p, :, o].cpu()
        if hd % 16:
            assert int(raw[..., hd:].max()) == 0                                  # padding
        got = raw[..., :hd].contiguous().view(torch.int8 if fmt == "i8" else torch.float8_e4m3fn).double()
        assert torch.equal(got, R.codes(x[here].cpu(), want_e, fmt))
        untouched = torch.ones(pages, page, dtype=torch.bool)
        untouched[p.cpu(), o.cpu()] = False
        assert int((c.cpu().permute(0, 2, 1, 3)[untouched] != 0xAB).sum()) == 0 and int(e.cpu().permute(0, 2, 1)[untouched].sum()) == 0
    k2, v2 = torch.full_like(k, 7.0), torch.full_like(v, 7.0)
    hip.cache_read(ck, cv, ek, ev, slots, k2, v2, **kw)
    for got, c, e in ((k2, ck, ek), (v2, cv, ev)):
        assert torch.equal(got[here].cpu(), R.decode(c[p, :, o][..., :hd], e[p, :, o], fmt).to(dt))
        assert bool((got[~here] == 7.0).all())


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("pairing", ["halves", "adjacent"])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,kv_heads,hd,sections", [(1, 2, 64, (8, 12, 12)), (90, 3, 24, (2, 5, 5)), (1100, 2, 128, (16, 24, 24)), (40, 4, 96, (4, 8, 12)),
                                                       (17, 2, 8, (2, 1, 1))])
def test_cache_write_turns_the_keys(rows, kv_heads, hd, sections, dt, pairing, fmt):
    """A stored key is within half a code's step of the turned key; the exponent is the rule's for a row as large as the turned one."""
    k, pos, freq = rotary_inputs(rows, kv_heads, hd, sum(sections), dt, hd + rows)
    v = cache_rows(rows, kv_heads, hd, dt, 2)
    page, pages = 32, -(-rows // 32)
    ck, cv, ek, ev = new_cache(pages, kv_heads, page, hd)
    slots = torch.arange(rows, device=DEV)
    kw = dict(rows=rows, kv_heads=kv_heads, hd=hd, page_size=page, fmt=FMT[fmt])
    hip.cache_write(k, v, ck, cv, ek, ev, slots, pos=pos, freq=freq, sections=sections, pairing=PAIR[pairing], **kw)
    want, size = R.rotate(k, pos, freq, sections, pairing)
    p, o = slots // page, slots % page
    e = ek[p, :, o].cpu().long()
    d = R.ROTATION * size
    low, high = R.exponents(want * (1 - 1e-6), fmt), R.exponents(want * (1 + 1e-6), fmt)
    assert bool(((e >= low) & (e <= high)).all())
    scale = torch.exp2(e.double() - 127)[..., None]
    code = (want / scale).abs()
    step = torch.ones_like(code) if fmt == "i8" else torch.exp2(torch.floor(torch.log2(code.clamp_min(2.0 ** -6))) - 3)
    got = R.decode(ck[p, :, o][..., :hd], ek[p, :, o], fmt)
    within(got, want, step * scale / 2 * (1 + 1e-5) + d)
    assert torch.equal(ev[p, :, o].cpu().long(), R.exponents(v.cpu(), fmt))


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("dt", TYPES)
def test_cache_rows_with_infinities_and_nans_read_back_as_nan(dt, fmt):
    k = torch.randn((4, 2, 32), generator=gen(1)).to(dt).to(DEV)
    v = k.clone()
    k[0, 0, 5], k[1, 1, 31], v[2, 0, 0], v[3, 1, 7] = math.inf, math.nan, -math.inf, math.nan
    ck, cv, ek, ev = new_cache(1, 2, 16, 32)
    slots = torch.tensor([3, 0, 15, 7], device=DEV)
    kw = dict(rows=4, kv_heads=2, hd=32, page_size=16, fmt=FMT[fmt])
    hip.cache_write(k, v, ck, cv, ek, ev, slots, **kw)
    k2, v2 = torch.empty_like(k), torch.empty_like(v)
    hip.cache_read(ck, cv, ek, ev, slots, k2, v2, **kw)
    for x, y in ((k, k2), (v, v2)):
        assert torch.equal(torch.isnan(y).all(-1), ~torch.isfinite(x).all(-1)) and torch.equal(torch.isnan(y).any(-1), ~torch.isfinite(x).all(-1))


def test_cache_reads_empty_slots_as_zero_and_takes_strided_rows():
    hd, HK, page = 32, 2, 16
    buf = torch.randn((10, 200), generator=gen(2)).half().to(DEV)
    k, v = buf[:, 8:8 + 64], buf[:, 128:192]
    planes = new_cache(2, HK, page, hd)
    kw = dict(rows=10, kv_heads=HK, hd=hd, page_size=page, fmt=hip.CACHE_I8)
    slots = torch.arange(10, device=DEV) + 9
    hip.cache_write(k, v, *planes, slots, **kw)
    dense = new_cache(2, HK, page, hd)
    hip.cache_write(k.contiguous(), v.contiguous(), *dense, slots, **kw)
    assert all(torch.equal(a, b) for a, b in zip(planes, dense))
    out = torch.full((10, 160), 5.0, device=DEV)
    hip.cache_read(*planes, slots - 9, out[:, :64], out[:, 96:], **kw)
    back = torch.empty((10, 64), device=DEV), torch.empty((10, 64), device=DEV)
    hip.cache_read(*planes, slots, *back, **kw)
    assert torch.equal(out[9:, :64], back[0][:1]) and torch.equal(out[9:, 96:], back[1][:1])
    assert bool((out[:9, :64] == 0).all()) and bool((out[:9, 96:] == 0).all()) and bool((out[:, 64:96] == 5).all())


# ---- attention over the cache --------------------------------------------------------------------------------------------------
class Memory:
    """Sequences of the given key counts in a paged cache, garbage (NaN codes, odd exponents) in every slot that belongs to none."""

    def __init__(self, kv_len, kv_heads, hd, page, fmt, seed, spread=1.0):
        g = gen(seed)
        held = [-(-n // page) for n in kv_len]
        pages = sum(held) + 2
        self.kv_heads, self.hd, self.page, self.fmt = kv_heads, hd, page, fmt
        self.table = torch.full((len(kv_len), max(1, max(held))), -1, dtype=torch.int32)
        perm, at = torch.randperm(pages, generator=g).to(torch.int32), 0
        self.planes = new_cache(pages, kv_heads, page, hd, fill=0x7F)
        for e in self.planes[2:]:
            e.fill_(200)
        slots = []
        for s, n in enumerate(kv_len):
            self.table[s, :held[s]] = perm[at:at + held[s]]
            at += held[s]
            i = torch.arange(n)
            slots.append(self.table[s].long()[i // page] * page + i % page)
        slots = torch.cat(slots).to(DEV)
        rows = slots.numel()
        k = torch.randn((rows, kv_heads, hd), generator=g) * torch.exp(spread * torch.randn((rows, kv_heads, 1), generator=g) * 0.3)
        v = torch.randn((rows, kv_heads, hd), generator=g) * torch.exp(spread * torch.randn((rows, kv_heads, 1), generator=g)) + 0.2
        if rows:
            hip.cache_write(k.to(DEV), v.to(DEV), *self.planes, slots, rows=rows, kv_heads=kv_heads, hd=hd, page_size=page, fmt=FMT[fmt])
        self.slots, self.kv_len = slots, torch.tensor(kv_len, dtype=torch.int32)

    def attend(self, q, q_start, heads, visible=None, scale=None, out=None, **kw):
        q_start = torch.tensor(q_start, dtype=torch.int32)
        scale = self.hd ** -0.5 if scale is None else scale
        out = torch.full_like(q, 3.0) if out is None else out
        max_q = max(1, int((q_start[1:] - q_start[:-1]).max()))
        hip.cached_attention(q, out, *self.planes, self.table.to(DEV), self.kv_len.to(DEV), q_start.to(DEV), heads=heads, kv_heads=self.kv_heads,
                             hd=self.hd, page_size=self.page, fmt=FMT[self.fmt], max_q=max_q, scale=scale,
                             visible=None if visible is None else visible.to(DEV), **kw)
        want, tol = R.attend(q, *self.planes, self.table, self.kv_len, q_start, visible, heads, self.kv_heads, self.hd, self.page, self.fmt, scale)
        rows = ~torch.isnan(want).flatten(1).all(1)
        return out, want, tol, rows

    def check(self, q, q_start, heads, **kw):
        out, want, tol, rows = self.attend(q, q_start, heads, **kw)
        got = out.reshape(q.shape[0], heads, self.hd)
        within(got[rows.to(DEV)], want[rows], tol[rows])
        return out, want, rows


def queries(rows, heads, hd, dt, seed, size=1.0):
    return (torch.randn((rows, heads, hd), generator=gen(seed)) * size).to(dt).to(DEV)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("kv_len,q_len,heads,kv_heads,hd,page", [
    ([1], [1], 1, 1, 8, 16),                               # one key
    ([130], [1], 6, 6, 64, 1376),                          # one token
    ([700, 1, 33, 64], [1, 1, 1, 1], 8, 2, 64, 16),        # grouped heads, ragged lengths
    ([32] * 9, [1] * 9, 8, 8, 32, 32),                     # a temporal module's positions
    ([7, 40, 17], [2, 5, 3], 4, 4, 24, 16),                # a few tokens each
    ([300], [3], 16, 1, 128, 32),                          # all heads share one key head
    ([95, 257], [1, 4], 3, 3, 96, 48),
    ([90], [2], 2, 2, 48, 16),
    ([50], [1], 2, 1, 16, 16),
    ([129], [70], 2, 2, 64, 16),                           # many rows
    ([65, 200], [33, 129], 2, 1, 32, 64),
    ([300], [40], 1, 1, 128, 1376),
    ([140], [37], 2, 2, 96, 16),
    ([64], [64], 1, 1, 8, 16),
    ([1300, 700], [70, 100], 6, 2, 64, 64),                # several row blocks, the keys in parts
    ([2000, 40], [6, 4], 8, 2, 32, 32),
    ([1100], [140], 2, 2, 128, 16),
])
def test_attention_over_the_cache(kv_len, q_len, heads, kv_heads, hd, page, dt, fmt):
    m = Memory(kv_len, kv_heads, hd, page, fmt, 11)
    start = [0]
    for n in q_len:
        start.append(start[-1] + n)
    m.check(queries(start[-1], heads, hd, dt, 12), start, heads)


@pytest.mark.parametrize("fmt,dt", [("i8", torch.float16), ("e4m3", torch.bfloat16), ("i8", torch.float32)])
@pytest.mark.parametrize("q_len", [3, 50, 150])
def test_attention_sees_only_visible_keys(q_len, fmt, dt):
    """Causal by frames of seven tokens, rows that see nothing, limits beyond the length; NaN rows among the keys that a row must
    not see."""
    kv = q_len + 100
    m = Memory([kv, 40], 2, 64, 32, fmt, 21)
    visible = torch.tensor([min(kv, kv - q_len + (i // 7 + 1) * 7) for i in range(q_len)] + [10, 0, -5, 10 ** 9], dtype=torch.int32)
    q = queries(q_len + 4, 4, 64, dt, 22)
    out, want, rows = m.check(q, [0, q_len, q_len + 4], 4, visible=visible)
    assert bool((out[q_len + 1:q_len + 3] == 0).all())
    last = m.slots[kv - 1]                                  # the first sequence's last key becomes NaN: only rows that see it change
    bad = torch.full((1, 2, 64), math.nan, device=DEV)
    hip.cache_write(bad, bad, *m.planes, last[None], rows=1, kv_heads=2, hd=64, page_size=32, fmt=FMT[fmt])
    again = m.attend(q, [0, q_len, q_len + 4], 4, visible=visible)[0]
    sees = torch.tensor([n >= kv for n in visible.tolist()])
    sees[q_len:] = False
    assert bool(torch.isnan(again[sees.to(DEV)]).all()) and torch.equal(again[~sees.to(DEV)], out[~sees.to(DEV)])


@pytest.mark.parametrize("q_len", [1, 40])
@pytest.mark.parametrize("dt", TYPES)
def test_attention_of_a_visible_nan_row(dt, q_len):
    m = Memory([50], 1, 32, 16, "e4m3", 31)
    bad = torch.full((1, 1, 32), math.nan, device=DEV)
    good = torch.ones((1, 1, 32), device=DEV)
    hip.cache_write(good, bad, *m.planes, m.slots[20:21], rows=1, kv_heads=1, hd=32, page_size=16, fmt=hip.CACHE_E4M3)
    q = queries(q_len, 2, 32, dt, 32)
    out = m.attend(q, [0, q_len], 2)[0]
    assert bool(torch.isnan(out).all())                     # the value row is NaN, whatever its key


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("q_len,dt", [(1, torch.float16), (1, torch.float32), (5, torch.bfloat16), (40, torch.float16), (40, torch.float32)])
def test_attention_with_evicted_pages_and_empty_slots(q_len, dt, fmt):
    m = Memory([200, 90, 0, 31], 2, 64, 16, fmt, 41)
    m.table[0, 3], m.table[0, 12], m.table[1, 0] = -1, m.planes[0].shape[0], 2 ** 31 - 1      # outside the cache: hidden
    m.table[3] = -1                                                                            # nothing left
    m.planes[2].view(-1)[::5] = 0                                                              # empty slots in every page
    start = [0, q_len, 2 * q_len, 3 * q_len, 4 * q_len]
    out, want, rows = m.check(queries(4 * q_len, 4, 64, dt, 42), start, 4)
    assert bool((out[2 * q_len:] == 0).all())


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("q_len,dt", [(1, torch.float16), (2, torch.float32), (40, torch.bfloat16), (40, torch.float32)])
def test_attention_over_rows_of_very_different_sizes(q_len, dt, fmt):
    """Values whose exponents lie up to thirty octaves apart, zero rows among them, keys of all sizes."""
    m = Memory([150], 1, 32, 16, fmt, 51)
    g = gen(52)
    k = torch.randn((150, 1, 32), generator=g) * torch.exp2(torch.randint(-14, 1, (150, 1, 1), generator=g).float())
    v = torch.randn((150, 1, 32), generator=g) * torch.exp2(torch.randint(-15, 16, (150, 1, 1), generator=g).float())
    k[::11], v[::13], v[3] = 0, 0, 0
    hip.cache_write(k.to(DEV), v.to(DEV), *m.planes, m.slots, rows=150, kv_heads=1, hd=32, page_size=16, fmt=FMT[fmt])
    m.check(queries(q_len, 1, 32, dt, 53), [0, q_len], 1)


@pytest.mark.parametrize("size", [1e-6, 30.0, 3e4])
@pytest.mark.parametrize("q_len,dt", [(1, torch.float16), (1, torch.bfloat16), (3, torch.float32), (40, torch.bfloat16), (40, torch.float32)])
def test_attention_with_tiny_and_huge_queries(q_len, dt, size):
    m = Memory([120], 2, 64, 32, "i8", 61)
    q = queries(q_len, 2, 64, dt, 62, 1.0)
    q = (q.float() * size).clamp(-6e4, 6e4).to(dt)
    m.check(q, [0, q_len], 2, scale=0.125 / size)           # the products, not the operands, set the scores
    q[0] = 0                                                # a row of zeros weighs all keys alike
    m.check(q, [0, q_len], 2, scale=0.125 / size)


@pytest.mark.parametrize("q_len", [1, 30])
def test_attention_rows_of_no_sequence_and_strided_rows(q_len):
    m = Memory([70, 20], 2, 64, 16, "i8", 71)
    rows = 2 * q_len + 5
    buf = torch.randn((rows, 3 * 4 * 64), generator=gen(72)).half().to(DEV)
    out = torch.full((rows, 400), 9.0, dtype=torch.float16, device=DEV)
    start = [2, 2 + q_len, 2 + 2 * q_len]
    q = buf[:, 256:512]
    m.check(q.contiguous().view(rows, 4, 64), start, 4)
    dense = m.attend(q.contiguous().view(rows, 4, 64), start, 4)[0].reshape(rows, 256)
    hip.cached_attention(q, out[:, 64:320], *m.planes, m.table.to(DEV), m.kv_len.to(DEV), torch.tensor(start, dtype=torch.int32, device=DEV), heads=4,
                         kv_heads=2, hd=64, page_size=16, fmt=hip.CACHE_I8, max_q=q_len, scale=0.125)
    live = slice(2, 2 + 2 * q_len)
    assert torch.equal(out[live, 64:320], dense[live])
    assert bool((out[:2] == 9).all()) and bool((out[2 + 2 * q_len:] == 9).all()) and bool((out[:, :64] == 9).all()) and bool((out[:, 320:] == 9).all())
    # starts beyond the rows are cut to them, lengths beyond the table to it, rows beyond max_q stay as they were
    start2 = torch.tensor([0, q_len, 10 ** 9], dtype=torch.int32, device=DEV)
    out.fill_(9.0)
    hip.cached_attention(q, out[:, 64:320], *m.planes, m.table.to(DEV), torch.tensor([10 ** 9, -3], dtype=torch.int32, device=DEV), start2, heads=4,
                         kv_heads=2, hd=64, page_size=16, fmt=hip.CACHE_I8, max_q=q_len, scale=0.125)
    assert bool((out[q_len:2 * q_len, 64:320] == 0).all()) and bool((out[2 * q_len:] == 9).all())


@pytest.mark.parametrize("q_len,kv", [(1, 20000), (9, 6000), (64, 5000), (300, 1500)])
def test_attention_is_the_same_bits_from_run_to_run_and_under_graph_replay(q_len, kv):
    """The long axis is split over workgroups and joined in a fixed order; the workspace may hold anything."""
    m = Memory([kv], 2, 64, 64, "i8", 81)
    q = queries(q_len, 4, 64, torch.float16, 82)
    table, kv_len, start = m.table.to(DEV), m.kv_len.to(DEV), torch.tensor([0, q_len], dtype=torch.int32, device=DEV)
    shape = dict(heads=4, kv_heads=2, hd=64, page_size=64, fmt=hip.CACHE_I8, max_q=q_len)
    n = hip.cached_attention_work(m.planes[0], seqs=1, max_pages=table.shape[1], **shape)
    work = torch.full((max(n, 16),), 0xFF, dtype=torch.uint8, device=DEV)
    first, out = torch.empty_like(q), torch.empty_like(q)
    hip.cached_attention(q, first, *m.planes, table, kv_len, start, scale=0.125, work=work, **shape)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        hip.cached_attention(q, out, *m.planes, table, kv_len, start, scale=0.125, work=work, **shape)
    for i in range(3):
        work.fill_(0xFF if i else 0x7F)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first)
        q.copy_(queries(q_len, 4, 64, torch.float16, 90 + i))
        hip.cached_attention(q, first, *m.planes, table, kv_len, start, scale=0.125, **shape)
    if q_len == 1:
        m.check(q, [0, 1], 4)


# ---- norms around a block -------------------------------------------------------------------------------------------------------
# Statistics: sums of C terms in a tree of at most 40 fp32 additions, the root and the products after it: 48 roundings of 2^-24 of
# the terms' sizes.
NORM_ERROR = 48 * 2.0 ** -24


@pytest.mark.parametrize("post", ["none", "layer", "rms"])
@pytest.mark.parametrize("pre", ["none", "layer", "rms"])
@pytest.mark.parametrize("bt,yt", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32), (torch.float32, torch.float16)])
@pytest.mark.parametrize("rows,C,per", [(1, 4, 1), (7, 384, 3), (130, 1024, 64), (5, 1028, 5), (3, 2048, 2), (4, 4096, 1), (3, 5000, 3), (2, 8192, 1), (9, 200, 100)])
def test_gated_norm(rows, C, per, pre, post, bt, yt):
    g = gen(rows + C)
    groups = -(-rows // per)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    x, b = (r(rows, C) * 2 + 3).to(DEV), (r(rows, C) + 0.5).to(bt).to(DEV)
    vec = dict(post_w=1 + 0.2 * r(C), post_b=0.1 * r(C), gate=r(groups, C), pre_w=1 + 0.2 * r(C), pre_b=0.1 * r(C), mod_scale=0.3 * r(groups, C),
               mod_shift=r(groups, C))
    if rows == 7:
        vec = dict.fromkeys(vec)                            # none of them
    if rows == 9:
        vec["gate"] = vec["mod_shift"] = vec["post_b"] = vec["pre_b"] = None
    vec = {n: None if t is None else t.to(DEV) for n, t in vec.items()}
    x_out, y = torch.full_like(x, math.nan), torch.full((rows, C), math.nan, dtype=yt, device=DEV)
    kw = dict(rows=rows, C=C, post=NORM[post], pre=NORM[pre], resid_scale=0.8, rows_per_group=per, eps=1e-5, **vec)
    hip.gated_norm(x, b, x_out, y, **kw)
    want_x, want_y, size_x, size_y = R.gated_norm(x, b, post, resid_scale=0.8, pre=pre, per=per, eps=1e-5, **vec)
    within(x_out, want_x, NORM_ERROR * size_x, "x")
    within(y, want_y, NORM_ERROR * size_y + (0 if yt == torch.float32 else R.half_step(yt)) * (want_y.abs() + NORM_ERROR * size_y), "y")
    z = x.clone()
    y2 = torch.empty_like(y)
    hip.gated_norm(z, b, z, y2, **kw)                       # in place on the stream
    assert torch.equal(z, x_out) and torch.equal(y2, y)


@pytest.mark.parametrize("C", [384, 4100])
def test_gated_norm_of_the_stream_alone_the_update_alone_and_strided_rows(C):
    g = gen(C)
    rows = 6
    x, b = torch.randn((rows, C + 12), generator=g).to(DEV), torch.randn((rows, 2 * C), generator=g).half().to(DEV)
    w, gate = torch.randn(C, generator=g).to(DEV), torch.randn((1, C), generator=g).to(DEV)
    xs, bs = x[:, 4:4 + C], b[:, C:]
    out, y = torch.zeros((rows, C + 8), device=DEV), torch.zeros((rows, C + 4), dtype=torch.bfloat16, device=DEV)
    hip.gated_norm(xs, bs, out[:, 8:], y[:, :C], rows=rows, C=C, gate=gate, pre=hip.NORM_RMS, pre_w=w)
    d_out, d_y = torch.empty((rows, C), device=DEV), torch.empty((rows, C), dtype=torch.bfloat16, device=DEV)
    hip.gated_norm(xs.contiguous(), bs.contiguous(), d_out, d_y, rows=rows, C=C, gate=gate, pre=hip.NORM_RMS, pre_w=w)
    assert torch.equal(out[:, 8:], d_out) and torch.equal(y[:, :C], d_y) and bool((out[:, :8] == 0).all()) and bool((y[:, C:] == 0).all())
    only = torch.empty_like(d_out)
    hip.gated_norm(xs, bs, only, None, rows=rows, C=C, gate=gate, pre=hip.NORM_NONE)
    assert torch.equal(only, d_out)
    y3 = torch.empty_like(d_y)
    hip.gated_norm(d_out, None, None, y3, rows=rows, C=C, pre=hip.NORM_RMS, pre_w=w)
    assert torch.equal(y3, d_y)


def test_gated_norm_is_the_frameworks_layernorm_on_a_plain_stream():
    """With a LayerNorm and nothing else it computes what vda_layernorm does, to rounding."""
    x = torch.randn((50, 1024), generator=gen(1)).to(DEV)
    w, b = torch.randn(1024, generator=gen(2)).to(DEV), torch.randn(1024, generator=gen(3)).to(DEV)
    a, y = torch.empty_like(x), torch.empty_like(x)
    hip.layernorm(x, a, w, b, 50, 1024, 1e-6)
    hip.gated_norm(x, None, None, y, rows=50, C=1024, pre_w=w, pre_b=b, eps=1e-6)
    within(y, a.double().cpu(), 2 * NORM_ERROR * (x.abs().double().cpu().amax() * w.abs().double().cpu().amax() + 4))


# ---- calls at the ends of what is allowed ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("q_len", [1, 40])
@pytest.mark.parametrize("scale", [-0.2, 0.0])
def test_attention_with_a_negative_and_a_zero_scale(q_len, scale):
    """A negative scale prefers the keys that point away; 0 weighs all that are seen alike, and still nothing else."""
    table_pages = 1 if q_len == 1 else 300                  # (a long table of absent pages: the kernel for many rows)
    m = Memory([100, 33], 2, 64, 16, "i8", 101)
    m.table = torch.nn.functional.pad(m.table, (0, table_pages), value=-1)
    visible = torch.tensor([90] * q_len + [0] * q_len, dtype=torch.int32)
    out = m.check(queries(2 * q_len, 4, 64, torch.float16, 102), [0, q_len, 2 * q_len], 4, scale=scale, visible=visible)[0]
    assert bool((out[q_len:] == 0).all())


@pytest.mark.parametrize("q_len,heads,hd", [(1, 8, 128), (64, 8, 128), (40, 16, 96)])
def test_cache_rows_behind_4_gib(q_len, heads, hd):
    """Planes of more than 2^32 bytes: the pages in use are the last ones and the first."""
    kv_heads, page = 8, 64
    pages = (1 << 32) // (page * kv_heads * hip.cache_row_bytes(hd)) + 300
    planes = [torch.empty((pages, kv_heads, page, hip.cache_row_bytes(hd)), dtype=torch.uint8, device=DEV) for _ in range(2)]
    planes += [torch.zeros((pages, kv_heads, page), dtype=torch.uint8, device=DEV) for _ in range(2)]
    used = [pages - 1, 0, pages - 2, pages - 7, 1]
    n = 4 * page + 9
    i = torch.arange(n)
    slots = (torch.tensor(used)[i // page] * page + i % page).to(DEV)
    g = gen(111)
    k, v = (torch.randn((n, kv_heads, hd), generator=g).to(DEV) for _ in range(2))
    kw = dict(kv_heads=kv_heads, hd=hd, page_size=page, fmt=hip.CACHE_I8)
    hip.cache_write(k, v, *planes, slots, rows=n, **kw)
    k2, v2 = torch.empty_like(k), torch.empty_like(v)
    hip.cache_read(*planes, slots, k2, v2, rows=n, **kw)
    for x, y in ((k, k2), (v, v2)):
        e = R.exponents(x.cpu(), "i8")
        assert torch.equal(y.cpu().double(), R.codes(x.cpu(), e, "i8") * torch.exp2(e.double() - 127)[..., None])
    q = queries(q_len, heads, hd, torch.float16, 112)
    out = torch.empty_like(q)
    table = torch.full((1, 5 if q_len == 1 else 500), -1, dtype=torch.int32)
    table[0, :5] = torch.tensor(used)
    start, length = torch.tensor([0, q_len], dtype=torch.int32), torch.tensor([n], dtype=torch.int32)
    hip.cached_attention(q, out, *planes, table.to(DEV), length.to(DEV), start.to(DEV), heads=heads, max_q=q_len, scale=hd ** -0.5, **kw)
    small = [p[used].contiguous() for p in planes]           # the same rows in a small cache, for the reference
    table[0, :5] = torch.arange(5)
    want, tol = R.attend(q, *small, table, length, start, None, heads, kv_heads, hd, page, "i8", hd ** -0.5)
    within(out, want, tol)


@pytest.mark.parametrize("q_len,kv", [(1, 6000), (200, 6000)])
def test_attention_graphs_on_two_streams_with_workspaces_of_their_own(q_len, kv):
    """Two captured calls replayed side by side, with eager calls on a third stream between, give what one call alone gives."""
    m = Memory([kv], 2, 64, 64, "e4m3", 121)
    table, kv_len, start = m.table.to(DEV), m.kv_len.to(DEV), torch.tensor([0, q_len], dtype=torch.int32, device=DEV)
    shape = dict(heads=4, kv_heads=2, hd=64, page_size=64, fmt=hip.CACHE_E4M3, max_q=q_len)
    n = hip.cached_attention_work(m.planes[0], seqs=1, max_pages=table.shape[1], **shape)
    assert n > 0
    qs = [queries(q_len, 4, 64, torch.bfloat16, 122 + i) for i in range(3)]
    want = [torch.empty_like(q) for q in qs]
    for q, w in zip(qs, want):
        hip.cached_attention(q, w, *m.planes, table, kv_len, start, scale=0.125, **shape)
    torch.cuda.synchronize()
    outs, graphs, streams = [], [], [torch.cuda.Stream() for _ in range(3)]
    works = [torch.empty(n, dtype=torch.uint8, device=DEV) for _ in range(2)]
    for q, work in zip(qs, works):
        out, graph = torch.empty_like(q), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            hip.cached_attention(q, out, *m.planes, table, kv_len, start, scale=0.125, work=work, **shape)
        outs.append(out)
        graphs.append(graph)
    for _ in range(3):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            third = torch.empty_like(qs[2])
            hip.cached_attention(qs[2], third, *m.planes, table, kv_len, start, scale=0.125, **shape)
        torch.cuda.synchronize()
        for got, w in zip(outs + [third], want):
            assert torch.equal(got, w)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("q_len,kv,table_pages", [(1, 40, 3), (5, 700, 44), (3, 6000, 375), (150, 700, 300)])
def test_attention_in_place_of_its_queries(q_len, kv, table_pages, dt):
    m = Memory([kv, 33], 2, 64, 16, "i8", 141)
    m.table = torch.nn.functional.pad(m.table, (0, table_pages - m.table.shape[1]), value=-1)
    q = queries(2 * q_len, 4, 64, dt, 142)
    start = torch.tensor([0, q_len, 2 * q_len], dtype=torch.int32, device=DEV)
    kw = dict(heads=4, kv_heads=2, hd=64, page_size=16, fmt=hip.CACHE_I8, max_q=q_len, scale=0.125)
    out = torch.empty_like(q)
    hip.cached_attention(q, out, *m.planes, m.table.to(DEV), m.kv_len.to(DEV), start, **kw)
    hip.cached_attention(q, q, *m.planes, m.table.to(DEV), m.kv_len.to(DEV), start, **kw)
    assert torch.equal(q, out)


# ---- the operators together ----------------------------------------------------------------------------------------------------------
def product_check(got, a, w):
    """A product of 16-bit operands with fp32 sums, rounded to got's type."""
    a, w = a.double().cpu(), w.double().cpu()
    want, size = a @ w.t(), a.abs() @ w.abs().t()
    e = (a.shape[1] + 8) * 2.0 ** -24 * size
    within(got, want, e + R.half_step(got.dtype) * (want.abs() + e), "product")


@pytest.mark.parametrize("dt,fmt,tokens,table_pages,pairing", [(torch.bfloat16, "i8", 20, 3, "halves"), (torch.float16, "e4m3", 33, 200, "adjacent"), (torch.float16, "i8", 1, 3, "halves")])
def test_a_block_over_a_memory_of_frames(dt, fmt, tokens, table_pages, pairing):
    """Two streams pass frame after frame through norm, projections, rotation, the cache, attention over the last three frames, the
    output projection and the norms around it, with the oldest page given to the new frame; every step is held to its
    definition on what the step before it left.  The last frame again on a stream of its own and as a captured graph: the same bits."""
    streams, C, heads, kv_heads, hd, page, held = 2, 256, 4, 2, 64, 48, 3
    rows, qw, kw_ = streams * tokens, heads * hd, kv_heads * hd
    g = gen(131)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    w_in, w_out = (r(qw + 2 * kw_, C) / 16).to(dt).to(DEV), (r(C, qw) / 16).to(dt).to(DEV)
    freq = (torch.rand(hd // 2, generator=g, dtype=torch.float64)).to(DEV)
    vec = {n: t.to(DEV) for n, t in dict(post_w=1 + 0.1 * r(C), gate=r(streams, C), pre_w=1 + 0.1 * r(C), mod_scale=0.2 * r(streams, C), mod_shift=0.1 * r(streams, C)).items()}
    before = dict(rows=rows, C=C, pre=hip.NORM_RMS, pre_w=vec["pre_w"], mod_scale=vec["mod_scale"], mod_shift=vec["mod_shift"], rows_per_group=tokens)
    after = dict(rows=rows, C=C, post=hip.NORM_RMS, post_w=vec["post_w"], gate=vec["gate"], pre=hip.NORM_LAYER, rows_per_group=tokens)
    planes = new_cache(streams * held, kv_heads, page, hd)
    shape = dict(kv_heads=kv_heads, hd=hd, page_size=page, fmt=FMT[fmt])
    turn = dict(sections=(8, 12, 12), pairing=PAIR[pairing])
    table = torch.full((streams, table_pages), -1, dtype=torch.int32, device=DEV)
    kv_len, start = torch.zeros(streams, dtype=torch.int32, device=DEV), torch.arange(streams + 1, dtype=torch.int32, device=DEV) * tokens
    slots, pos, x = torch.empty(rows, dtype=torch.int64, device=DEV), torch.empty((rows, 3), dtype=torch.int32, device=DEV), torch.empty((rows, C), device=DEV)
    n = hip.cached_attention_work(planes[0], seqs=streams, max_pages=table_pages, max_q=tokens, heads=heads, **shape)
    work = torch.empty(max(n, 16), dtype=torch.uint8, device=DEV)

    def step():
        y, packed, att, b = (torch.empty((rows, w), dtype=dt, device=DEV) for w in (C, qw + 2 * kw_, qw, C))
        x_out, z = torch.empty_like(x), torch.empty((rows, C), dtype=dt, device=DEV)
        hip.gated_norm(x, None, None, y, **before)
        hip.gemm(y, w_in, packed, M=rows, N=qw + 2 * kw_, K=C, lda=C, ldc=qw + 2 * kw_)
        flat = packed.clone()
        q, k, v = packed[:, :qw], packed[:, qw:qw + kw_], packed[:, qw + kw_:]
        hip.rotary_axes(q, q, pos, freq, rows=rows, heads=heads, hd=hd, **turn)
        hip.cache_write(k, v, *planes, slots, rows=rows, pos=pos, freq=freq, **turn, **shape)
        hip.cached_attention(q, att, *planes, table, kv_len, start, heads=heads, max_q=tokens, scale=hd ** -0.5, work=work, **shape)
        hip.gemm(att, w_out, b, M=rows, N=C, K=qw, lda=qw, ldc=C)
        hip.gated_norm(x, b, x_out, z, **after)
        return y, flat, packed, att, b, x_out, z

    for f in range(5):
        # a stream's pages in the order of their frames; place f % held is the newest frame's, the oldest one's before
        at = [s * held + (f - i) % held for s in range(streams) for i in reversed(range(min(f + 1, held)))]
        table[:, :min(f + 1, held)] = torch.tensor(at, dtype=torch.int32).reshape(streams, -1).to(DEV)
        full = min(f, held - 1)                                              # older frames; their unused places are empty slots
        kv_len.fill_(full * page + tokens)
        t = torch.arange(tokens)
        slots.copy_(torch.cat([(s * held + f % held) * page + t for s in range(streams)]))
        pos.copy_(torch.stack([torch.full((tokens,), 30 * f), t // 7, t % 7], 1).repeat(streams, 1))
        x.copy_(r(rows, C))
        y, flat, packed, att, b, x_out, z = step()
        rounding = lambda want, e: e + R.half_step(dt) * (want.abs() + e)  # noqa: E731
        _, want, _, size = R.gated_norm(x, None, "none", None, None, None, 1.0, "rms", vec["pre_w"], None, vec["mod_scale"], vec["mod_shift"], tokens, 1e-6)
        within(y, want, rounding(want, NORM_ERROR * size), "first norm")
        product_check(flat, y, w_in)
        rotary_check(packed[:, :qw].reshape(rows, heads, hd), flat[:, :qw].reshape(rows, heads, hd), pos, freq, turn["sections"], pairing)
        assert torch.equal(packed[:, qw:], flat[:, qw:])
        p, o = slots // page, slots % page
        want, size = R.rotate(flat[:, qw:qw + kw_].reshape(rows, kv_heads, hd), pos, freq, turn["sections"], pairing)
        scale = torch.exp2(planes[2][p, :, o].cpu().double() - 127)[..., None]
        code_step = torch.ones_like(want) if fmt == "i8" else torch.exp2(torch.floor(torch.log2((want / scale).abs().clamp_min(2.0 ** -6))) - 3)
        within(R.decode(planes[0][p, :, o][..., :hd], planes[2][p, :, o], fmt), want, code_step * scale / 2 * (1 + 1e-5) + R.ROTATION * size, "keys")
        want, tol = R.attend(packed[:, :qw].reshape(rows, heads, hd), *planes, table.cpu(), kv_len, start, None, heads, kv_heads, hd, page, fmt, hd ** -0.5)
        within(att.reshape(rows, heads, hd), want, tol, "attention")
        product_check(b, att, w_out)
        want_x, want, size_x, size = R.gated_norm(x, b, "rms", vec["post_w"], None, vec["gate"], 1.0, "layer", None, None, None, None, tokens, 1e-6)
        within(x_out, want_x, NORM_ERROR * size_x, "stream")
        within(z, want, rounding(want, NORM_ERROR * size), "last norm")

    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = step()
    torch.cuda.synchronize()
    assert torch.equal(again[-1], z) and torch.equal(again[-2], x_out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for i in range(3):
        captured[-1].zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured[-1], z) and torch.equal(captured[-2], x_out)
        step()                                                              # eager work between the replays
        torch.cuda.synchronize()


# ---- what a row does not see, and what it sees but does not weigh --------------------------------------------------------------------
WIDE = [(torch.float16, "i8"), (torch.bfloat16, "e4m3"), (torch.float32, "i8"), (torch.float32, "e4m3")]


def store(m, at, k, v):
    """k and v ([rows, hd], for every key head) into the slots of the keys ``at``, counted over the sequences."""
    rows = len(at)
    wide = lambda x: x[:, None].expand(rows, m.kv_heads, m.hd).contiguous().to(DEV)  # noqa: E731
    hip.cache_write(wide(k), wide(v), *m.planes, m.slots[at], rows=rows, kv_heads=m.kv_heads, hd=m.hd, page_size=m.page, fmt=FMT[m.fmt])


def unseen_keys_have_no_effect(q_len, kv, first, table_pages, size, hd, dt, fmt, same_bits):
    """Every row but the last ends before key ``first``; keys from there on then become finite and very large, in the tile of the last key
    that the rows see and behind it: no bit of those rows changes, or (the kernel for many rows, whose rows move their references together and
    which takes another form where exponents lie far apart) they stay within the bound of what they see."""
    m = Memory([kv], 2, hd, 16, fmt, 151)
    m.table = torch.nn.functional.pad(m.table, (0, max(0, table_pages - m.table.shape[1])), value=-1)
    visible = torch.full((q_len,), first, dtype=torch.int32)
    visible[:q_len // 2] -= torch.arange(q_len // 2, dtype=torch.int32) % 5
    visible[-1] = kv
    q = queries(q_len, 4, hd, dt, 152)
    out, want, rows = m.check(q, [0, q_len], 4, visible=visible)
    late = list(range(first, kv))
    one = torch.ones((len(late), hd))
    for k, v in ((one, one * size), (one * size, one), (-one * size, one * size)):
        store(m, late, k, v)
        again, want, tol, _ = m.attend(q, [0, q_len], 4, visible=visible)
        within(again[:-1], want[:-1], tol[:-1])
        assert not same_bits or torch.equal(again[:-1], out[:-1])


def keys_without_weight_have_no_effect(q_len, table_pages, dt, fmt, hd=64):
    """A key that points far away from every query has weight 0, however large it and its value are: the rows are held to the bound of
    the memory without it."""
    m = Memory([90], 1, hd, 16, fmt, 161)
    m.table = torch.nn.functional.pad(m.table, (0, max(0, table_pages - m.table.shape[1])), value=-1)
    q = queries(q_len, 2, hd, dt, 162)
    q[..., 0] = q[..., 0].abs() + 1
    at = 37
    page, place = int(m.slots[at]) // 16, int(m.slots[at]) % 16
    m.planes[2][page, :, place] = 0
    start = torch.tensor([0, q_len], dtype=torch.int32)
    want, tol = R.attend(q, *m.planes, m.table, m.kv_len, start, None, 2, 1, hd, 16, fmt, hd ** -0.5)
    away = torch.zeros((1, hd))
    for far, size in ((-2.0 ** 36, 1.0), (-2.0 ** 36, 2.0 ** 40), (-2.0 ** 14, 2.0 ** 40)):
        away[0, 0] = far
        store(m, [at], away, torch.ones((1, hd)) * size)
        within(m.attend(q, [0, q_len], 2)[0], want, tol, f"key {far:.0e}, value {size:.0e}")


def large_values_of_small_weight_count(q_len, table_pages, dt, fmt, hd=32):
    """Values up to 2^40 times larger than the rest, on keys whose weights are as much smaller: both parts make up the output."""
    m = Memory([200], 1, hd, 16, fmt, 171)
    m.table = torch.nn.functional.pad(m.table, (0, max(0, table_pages - m.table.shape[1])), value=-1)
    g = gen(172)
    octaves = torch.randint(0, 41, (60, 1), generator=g).float()
    k, v = torch.randn((60, hd), generator=g) * 0.1, torch.randn((60, hd), generator=g) * torch.exp2(octaves)
    k[:, 0] = -(octaves[:, 0] * math.log(2.0) + 2) * hd ** 0.5
    store(m, list(range(3, 183, 3)), k, v)
    q = queries(q_len, 2, hd, dt, 173, 0.3)
    q[..., 0] = 1.0
    m.check(q, [0, q_len], 2)


@pytest.mark.parametrize("dt,fmt", WIDE)
@pytest.mark.parametrize("size", [2.0 ** 12, 2.0 ** 20, 2.0 ** 40])
@pytest.mark.parametrize("q_len,kv,first", [(3, 90, 71), (50, 150, 100), (150, 110, 80), (4, 3000, 1300)])
def test_attention_few_rows_unseen_keys_have_no_effect(q_len, kv, first, size, dt, fmt):
    unseen_keys_have_no_effect(q_len, kv, first, 0, size, 64, dt, fmt, True)


@pytest.mark.parametrize("dt,fmt", WIDE)
@pytest.mark.parametrize("q_len", [1, 40])
def test_attention_few_rows_keys_without_weight_have_no_effect(q_len, dt, fmt):
    keys_without_weight_have_no_effect(q_len, 0, dt, fmt)


@pytest.mark.parametrize("dt,fmt", [(torch.bfloat16, "i8"), (torch.bfloat16, "e4m3"), (torch.float32, "i8"), (torch.float32, "e4m3")])
@pytest.mark.parametrize("q_len,table_pages", [(1, 0), (40, 0), (1, 400)])
def test_attention_few_rows_large_values_of_small_weight_count(q_len, table_pages, dt, fmt):
    large_values_of_small_weight_count(q_len, table_pages, dt, fmt)


@pytest.mark.parametrize("dt,fmt", [(torch.float16, "i8"), (torch.bfloat16, "e4m3"), (torch.float32, "i8")])
@pytest.mark.parametrize("hd", [8, 24, 40, 48, 96, 128])
def test_attention_few_rows_parts_joined_for_every_head_size(hd, dt, fmt):
    """3000 keys in parts, heads that fill their padded size and heads that do not."""
    m = Memory([3000, 40], 2, hd, 16, fmt, 181)
    shape = dict(kv_heads=2, hd=hd, page_size=16, fmt=FMT[fmt])
    assert hip.cached_attention_work(m.planes[0], seqs=2, max_pages=m.table.shape[1], max_q=2, heads=4, **shape) > 0
    m.check(queries(3, 4, hd, dt, 182), [0, 2, 3], 4)


@pytest.mark.parametrize("dt,fmt", WIDE)
@pytest.mark.parametrize("size", [2.0 ** 3, 2.0 ** 12, 2.0 ** 20, 2.0 ** 40])
@pytest.mark.parametrize("q_len,kv,first,hd", [(150, 300, 200, 64), (70, 2000, 1100, 64), (300, 500, 130, 128)])
def test_attention_many_rows_unseen_keys_have_no_effect(q_len, kv, first, hd, size, dt, fmt):
    unseen_keys_have_no_effect(q_len, kv, first, 300, size, hd, dt, fmt, False)


@pytest.mark.parametrize("dt,fmt", WIDE)
@pytest.mark.parametrize("q_len", [40, 200])
def test_attention_many_rows_keys_without_weight_have_no_effect(q_len, dt, fmt):
    keys_without_weight_have_no_effect(q_len, 300, dt, fmt)


@pytest.mark.parametrize("dt,fmt", [(torch.bfloat16, "i8"), (torch.bfloat16, "e4m3"), (torch.float32, "i8"), (torch.float32, "e4m3")])
def test_attention_many_rows_large_values_of_small_weight_count(dt, fmt):
    large_values_of_small_weight_count(40, 300, dt, fmt)


@pytest.mark.parametrize("dt,fmt", WIDE)
@pytest.mark.parametrize("q_len,kv,hd", [(40, 150, 32), (150, 700, 64), (33, 1200, 96), (130, 400, 128)])
def test_attention_many_rows_over_rows_of_very_different_sizes(q_len, kv, hd, dt, fmt):
    """The kernel for many rows, which a long table selects: keys and values up to thirty octaves apart, rows of zeros among both, evicted
    pages; all keys seen, and a causal mask whose later keys are up to thirty octaves larger than the ones that every row sees."""
    for growing in (False, True):
        m = Memory([kv], 1, hd, 16, fmt, 191)
        g = gen(192)
        late = torch.arange(kv) >= kv - q_len
        k, v = torch.randn((kv, hd), generator=g), torch.randn((kv, hd), generator=g)
        if growing:
            k[late] *= torch.exp2(torch.randint(-8, 2, (q_len, 1), generator=g).float())
            v[late] *= torch.exp2(torch.randint(0, 31, (q_len, 1), generator=g).float())
        else:
            k *= torch.exp2(torch.randint(-14, 1, (kv, 1), generator=g).float())
            v *= torch.exp2(torch.randint(-15, 16, (kv, 1), generator=g).float())
            k[::11], v[::13], v[3] = 0, 0, 0
        store(m, list(range(kv)), k, v)
        m.table = torch.nn.functional.pad(m.table, (0, 300), value=-1)
        m.table[0, 2] = -1
        visible = (torch.arange(q_len) + kv - q_len + 1).int() if growing else None
        out, want, tol, _ = m.attend(queries(q_len, 2, hd, dt, 193), [0, q_len], 2, visible=visible)
        # what lies beyond half a step above fp16's largest number is infinite in fp16; at the border either side is right
        border = torch.finfo(dt).max * (1 + R.half_step(dt) / 2)
        beyond, border = want.abs() - tol >= border, (want.abs() + tol >= border) & (want.abs() - tol < border)
        got = out.double().cpu()
        assert torch.equal(got[beyond], want[beyond].sign() * math.inf)
        fine = ~beyond & ~border
        within(got[fine], want[fine], tol[fine])


@pytest.mark.parametrize("dt,fmt", [(torch.bfloat16, "i8"), (torch.bfloat16, "e4m3"), (torch.float32, "i8"), (torch.float32, "e4m3")])
@pytest.mark.parametrize("size", [1e-25, 1e-8, 1e34])
@pytest.mark.parametrize("q_len,kv,table_pages", [(1, 50, 0), (2, 6000, 0), (150, 200, 300), (70, 3000, 300)])
def test_attention_with_tiny_and_huge_values(q_len, kv, table_pages, size, dt, fmt):
    """Values near the ends of fp32's range, in the few-row kernel and in the one for many rows, in one part and in several."""
    m = Memory([kv], 1, 32, 16, fmt, 201)
    m.table = torch.nn.functional.pad(m.table, (0, max(0, table_pages - m.table.shape[1])), value=-1)
    g = gen(202)
    k, v = torch.randn((kv, 32), generator=g), torch.randn((kv, 32), generator=g)
    store(m, list(range(kv)), k, v * size)
    m.check(queries(q_len, 1, 32, dt, 203), [0, q_len], 1)


@pytest.mark.parametrize("dt,fmt", WIDE)
@pytest.mark.parametrize("size", [0.0, 1e-37])
@pytest.mark.parametrize("q_len,kv,table_pages", [(1, 6000, 0), (9, 700, 0), (70, 3000, 300), (200, 1500, 300)])
def test_attention_parts_whose_values_are_zeros_join_parts_whose_values_are_not(q_len, kv, table_pages, size, dt, fmt):
    """A part of the key axis without any value to speak of weighs in the sum of probabilities as every other."""
    m = Memory([kv], 1, 32, 16, fmt, 211)
    m.table = torch.nn.functional.pad(m.table, (0, max(0, table_pages - m.table.shape[1])), value=-1)
    g = gen(212)
    k, v = torch.randn((kv, 32), generator=g), torch.randn((kv, 32), generator=g)
    v[:kv // 2] *= size
    store(m, list(range(kv)), k, v)
    m.check(queries(q_len, 1, 32, dt, 213), [0, q_len], 1)


@pytest.mark.parametrize("dt,fmt", WIDE)
@pytest.mark.parametrize("spread", [0, 20])
@pytest.mark.parametrize("q_len,kv", [(40, 150), (150, 1300)])
def test_attention_many_rows_nan_rows_empty_slots_and_evicted_pages(q_len, kv, spread, dt, fmt):
    """The kernel for many rows, in its form for neighbouring exponents and in the one for others: a NaN row is seen by the rows that reach
    it, and by no other; empty slots and absent pages by none."""
    m = Memory([kv, 33], 2, 64, 16, fmt, 221)
    g = gen(222)
    v = torch.randn((kv, 64), generator=g) * torch.exp2(torch.randint(-spread // 2, spread // 2 + 1, (kv, 1), generator=g).float())
    store(m, list(range(kv)), torch.randn((kv, 64), generator=g), v)
    m.planes[2].view(-1)[::7] = 0
    m.table = torch.nn.functional.pad(m.table, (0, 300), value=-1)
    m.table[0, 4], m.table[0, 5] = -1, m.planes[0].shape[0]
    start = [0, q_len, q_len + 3]
    visible = torch.cat([torch.arange(q_len) + kv - q_len + 1, torch.tensor([33, 0, 20])]).int()
    q = queries(q_len + 3, 4, 64, dt, 223)
    out, want, rows = m.check(q, start, 4, visible=visible)
    assert bool((out[q_len + 1] == 0).all())
    at = kv - q_len // 2
    for k, v in ((math.nan, 1.0), (1.0, math.inf)):
        store(m, [at], torch.full((1, 64), k), torch.full((1, 64), v))
        again, want, tol, _ = m.attend(q, start, 4, visible=visible)
        sees = visible > at
        sees[q_len:] = False
        assert bool(torch.isnan(again[sees.to(DEV)]).all())
        within(again[~sees.to(DEV)], want[~sees], tol[~sees])
