"""What the wrappers and the C entries of the rotary, cache, attention and norm operators refuse, before anything is launched, and
their argument structs against the header."""
import ctypes
import os
import subprocess

import pytest
import torch

from video_depth_anything import hip

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EINVAL, ESHAPE = -1, -2
f16, f32, f64, u8, i32, i64 = torch.float16, torch.float32, torch.float64, torch.uint8, torch.int32, torch.int64


@pytest.fixture
def recorded(monkeypatch):
    """The wrappers with the library replaced by a recorder: what reaches the C ABI."""
    calls = []

    class Recorder:
        def __getattr__(self, name):
            return lambda *a: calls.append(name) or 0

    monkeypatch.setattr(hip, "lib", lambda: Recorder())
    monkeypatch.setattr(hip, "_dev", lambda *ts: None)
    monkeypatch.setattr(hip, "_current_device", lambda: -1)             # get_device() of a CPU tensor
    monkeypatch.setattr(hip, "_stream", lambda: None)
    return calls


def test_tensors_of_another_device_or_the_cpu_are_refused(monkeypatch):
    x = torch.zeros(4, 64, dtype=f16)
    with pytest.raises(RuntimeError, match="device tensors only"):
        hip.gated_norm(x.float(), None, None, x, rows=4, C=64)
    monkeypatch.setattr(hip, "_dev", lambda *ts: None)
    monkeypatch.setattr(hip, "_current_device", lambda: 0)
    with pytest.raises(ValueError, match="current device is 0"):
        hip.gated_norm(x.float(), None, None, x, rows=4, C=64)


def test_rotary_wrapper_refusals(recorded):
    x, pos, freq = torch.zeros(5, 128, dtype=f16), torch.zeros(5, 3, dtype=i32), torch.zeros(16, dtype=f64)
    kw = dict(rows=5, heads=2, hd=64, sections=(4, 6, 6))
    hip.rotary_axes(x, x, pos, freq, **kw)
    hip.rotary_axes(x, x.clone(), pos.float(), freq, **kw)
    assert len(recorded) == 2
    for bad, error, match in ((dict(x=x.float()), TypeError, "share"), (dict(pos=pos.long()), TypeError, "int32"), (dict(freq=freq.float()), TypeError, "float64"),
                              (dict(pos=pos[:4].clone()), ValueError, "pos holds"), (dict(freq=freq[:15].clone()), ValueError, "freq holds"),
                              (dict(pos=pos.t().contiguous().t()), ValueError, "dense"), (dict(out=x[:4].clone()), ValueError, "out holds"),
                              (dict(x=torch.zeros(5, 256, dtype=f16)[:, ::2]), ValueError, "not dense"), (dict(rows=6, pos=torch.zeros(6, 3, dtype=i32)), ValueError, "x holds")):
        args = {**dict(x=x, out=x, pos=pos, freq=freq), **kw, **bad}
        with pytest.raises(error, match=match):
            hip.rotary_axes(args.pop("x"), args.pop("out"), args.pop("pos"), args.pop("freq"), **args)
    assert len(recorded) == 2


def planes(pages=3, heads=2, page=16, hd=24):
    return [torch.zeros(pages, heads, page, hip.cache_row_bytes(hd), dtype=u8) for _ in "kv"] + [torch.zeros(pages, heads, page, dtype=u8) for _ in "kv"]


def test_cache_wrapper_refusals(recorded):
    k, v, slots = torch.zeros(5, 48, dtype=f16), torch.zeros(5, 48, dtype=f16), torch.zeros(5, dtype=i64)
    pos, freq = torch.zeros(5, 3, dtype=i32), torch.zeros(12, dtype=f64)
    kw = dict(rows=5, kv_heads=2, hd=24, page_size=16, fmt=hip.CACHE_I8)
    p = planes()
    hip.cache_write(k, v, *p, slots, **kw)
    hip.cache_write(k, v, *p, slots, pos=pos, freq=freq, sections=(4, 4, 4), **kw)
    hip.cache_read(*p, slots, k, v, **kw)
    assert recorded == ["vda_cache_write", "vda_cache_write", "vda_cache_read"]
    for bad, error, match in ((dict(v=v.float()), TypeError, "share"), (dict(slots=slots.int()), TypeError, "int64"), (dict(slots=slots[:4].clone()), ValueError, "slots holds"),
                              (dict(slots=torch.zeros(10, dtype=i64)[::2]), ValueError, "dense"), (dict(v=v[:4].clone()), ValueError, "v holds"),
                              (dict(k=torch.zeros(4, 48, dtype=f16)), ValueError, "k holds"), (dict(kv_heads=3), ValueError, "cache plane")):
        for name in ("write", "read"):
            a = {**dict(k=k, v=v, slots=slots), **kw, **bad}
            k_, v_, s_ = a.pop("k"), a.pop("v"), a.pop("slots")
            with pytest.raises(error, match=match):
                hip.cache_write(k_, v_, *p, s_, **a) if name == "write" else hip.cache_read(*p, s_, k_, v_, **a)
    for i in range(4):                                                  # a plane of another type, shape or order
        for bad in (p[i].to(torch.int8), p[i][:2], p[i].transpose(0, 1).contiguous().transpose(0, 1), p[i][..., :-1].contiguous()):
            with pytest.raises((TypeError, ValueError), match="cache plane"):
                hip.cache_write(k, v, *p[:i], bad, *p[i + 1:], slots, **kw)
    for part in (dict(pos=pos), dict(pos=pos, freq=freq), dict(sections=(4, 4, 4))):
        with pytest.raises(ValueError, match="come together"):
            hip.cache_write(k, v, *p, slots, **part, **kw)
    assert len(recorded) == 3


def test_attention_wrapper_refusals(recorded):
    p = planes()
    q = torch.zeros(6, 4, 24, dtype=f16)
    table, kv_len, start, seen = torch.zeros(2, 3, dtype=i32), torch.zeros(2, dtype=i32), torch.zeros(3, dtype=i32), torch.zeros(6, dtype=i32)
    kw = dict(heads=4, kv_heads=2, hd=24, page_size=16, fmt=hip.CACHE_E4M3, max_q=3, scale=0.2)
    hip.cached_attention(q, q.clone(), *p, table, kv_len, start, visible=seen, **kw)
    assert recorded == ["vda_cached_attention_work", "vda_cached_attention"]
    for bad, error, match in ((dict(out=q.float()), TypeError, "share"), (dict(table=table.long()), TypeError, "int32"), (dict(seen=seen[:5].clone()), ValueError, "visible holds"),
                              (dict(table=torch.zeros(3, 2, dtype=i32).t()), ValueError, "dense"), (dict(start=start[:2]), ValueError, "belong"),
                              (dict(kv_len=torch.zeros(3, dtype=i32)), ValueError, "belong"), (dict(out=q[:5].clone()), ValueError, "out holds"),
                              (dict(q=torch.zeros(6, 4, 48, dtype=f16)[..., ::2]), ValueError, "not dense")):
        a = {**dict(q=q, out=q.clone(), table=table, kv_len=kv_len, start=start, seen=seen), **bad}
        with pytest.raises(error, match=match):
            hip.cached_attention(a["q"], a["out"], *p, a["table"], a["kv_len"], a["start"], visible=a["seen"], **kw)


def test_attention_wrapper_refuses_a_small_workspace(recorded, monkeypatch):
    class Needs:
        vda_cached_attention_work = staticmethod(lambda *a: 4096)
        vda_cached_attention = staticmethod(lambda *a: recorded.append("vda_cached_attention") or 0)

    monkeypatch.setattr(hip, "lib", lambda: Needs)
    p, q = planes(), torch.zeros(1, 4, 24, dtype=f16)
    one = torch.zeros(1, 3, dtype=i32), torch.zeros(1, dtype=i32), torch.zeros(2, dtype=i32)
    kw = dict(heads=4, kv_heads=2, hd=24, page_size=16, fmt=hip.CACHE_E4M3, max_q=1, scale=0.2)
    hip.cached_attention(q, q.clone(), *p, *one, work=torch.zeros(4096, dtype=u8), **kw)
    with pytest.raises(ValueError, match="work holds 4095"):
        hip.cached_attention(q, q.clone(), *p, *one, work=torch.zeros(4095, dtype=u8), **kw)
    assert recorded == ["vda_cached_attention"]


def test_norm_wrapper_refusals(recorded):
    x, b, w = torch.zeros(6, 32), torch.zeros(6, 32, dtype=f16), torch.zeros(32)
    gate = torch.zeros(3, 32)
    kw = dict(rows=6, C=32, rows_per_group=2)
    hip.gated_norm(x, b, x, b.clone(), gate=gate, pre_w=w, **kw)
    assert recorded == ["vda_gated_norm"]
    for bad, error, match in ((dict(x=x.half()), TypeError, "fp32"), (dict(gate=gate[:2].clone()), ValueError, "gate holds"), (dict(gate=gate.half()), TypeError, "gate has to be torch.float32"),
                              (dict(gate=torch.zeros(3, 64)[:, ::2]), ValueError, "dense"), (dict(pre_w=w[:31].clone()), ValueError, "pre_w holds"),
                              (dict(b=b.to(i32)), TypeError, "b and y"), (dict(y=b[:5].clone()), ValueError, "y holds"), (dict(rows_per_group=0), ValueError, "positive"),
                              (dict(x_out=x[:5].clone()), ValueError, "x_out holds")):
        a = {**dict(x=x, b=b, x_out=x, y=b.clone(), gate=gate, pre_w=w), **kw, **bad}
        with pytest.raises(error, match=match):
            hip.gated_norm(a.pop("x"), a.pop("b"), a.pop("x_out"), a.pop("y"), **a)
    assert len(recorded) == 1


# ---- the C entries: every call below is refused before a launch (the pointers are never followed) -----------------------------------
A = 1 << 20                                                             # some 16-byte aligned address


def test_c_rotary_refusals():
    f = hip.lib().vda_rotary_axes
    good = dict(x=A, out=2 * A, pos=A, freq=A, rows=4, heads=2, hd=64, ldx=128, ldo=128, n_t=8, n_h=12, n_w=12, pairing=0, pos_float=0, dtype=hip.T_F16, stream=None)
    for bad, rc in ((dict(x=None), EINVAL), (dict(out=None), EINVAL), (dict(pos=None), EINVAL), (dict(freq=None), EINVAL), (dict(rows=0), EINVAL), (dict(heads=0), EINVAL),
                    (dict(dtype=0), EINVAL), (dict(dtype=7), EINVAL), (dict(pairing=2), EINVAL), (dict(n_t=-4, n_h=24), EINVAL), (dict(n_t=9), ESHAPE),
                    (dict(n_t=12), ESHAPE), (dict(n_t=0, n_h=0, n_w=0), ESHAPE), (dict(hd=60, n_t=0), ESHAPE), (dict(hd=264, ldx=528, ldo=528), ESHAPE),
                    (dict(ldx=120), ESHAPE), (dict(ldo=64), ESHAPE), (dict(x=A + 8), ESHAPE), (dict(ldx=129), ESHAPE), (dict(x=A + 4, out=A + 4), ESHAPE),
                    (dict(out=A, ldo=256), EINVAL), (dict(dtype=hip.T_F32, x=A + 8), ESHAPE), (dict(rows=1 << 50), ESHAPE)):
        assert f(*{**good, **bad}.values()) == rc, bad


def desc(**bad):
    return hip.CacheDesc(*{**dict(k=A, v=A, k_exp=A, v_exp=A, pages=4, page_size=32, kv_heads=2, hd=64, format=0), **bad}.values())


BAD_CACHES = [(dict(k=None), EINVAL), (dict(v=None), EINVAL), (dict(k_exp=None), EINVAL), (dict(v_exp=None), EINVAL), (dict(pages=0), EINVAL), (dict(page_size=-16), EINVAL),
              (dict(kv_heads=0), EINVAL), (dict(hd=0), EINVAL), (dict(format=2), EINVAL), (dict(hd=20), ESHAPE), (dict(hd=136), ESHAPE), (dict(page_size=24), ESHAPE),
              (dict(k=A + 8), ESHAPE), (dict(v_exp=A + 1), ESHAPE), (dict(pages=1 << 27), ESHAPE)]


def test_c_cache_refusals():
    w, r = hip.lib().vda_cache_write, hip.lib().vda_cache_read
    good = dict(k=A, v=A, slots=A, rows=4, ldk=128, ldv=128, dtype=hip.T_BF16, pos=A, freq=A, n_t=8, n_h=12, n_w=12, pairing=0, pos_float=0, stream=None)
    read = lambda a: (a["slots"], a["k"], a["v"], a["rows"], a["ldk"], a["ldv"], a["dtype"], None)  # noqa: E731
    for bad, rc in BAD_CACHES:
        assert w(ctypes.byref(desc(**bad)), *good.values()) == rc and r(ctypes.byref(desc(**bad)), *read(good)) == rc, bad
    for bad, rc in ((dict(k=None), EINVAL), (dict(v=None), EINVAL), (dict(slots=None), EINVAL), (dict(rows=0), EINVAL), (dict(dtype=0), EINVAL), (dict(ldk=120), ESHAPE),
                    (dict(ldv=127), ESHAPE), (dict(ldv=129), ESHAPE), (dict(k=A + 8), ESHAPE), (dict(rows=1 << 50), ESHAPE)):
        a = {**good, **bad}
        assert w(ctypes.byref(desc()), *a.values()) == rc and r(ctypes.byref(desc()), *read(a)) == rc, bad
    for bad, rc in ((dict(pos=None), EINVAL), (dict(freq=None), EINVAL), (dict(pairing=5), EINVAL), (dict(n_t=9), ESHAPE), (dict(n_t=12), ESHAPE), (dict(n_w=-4), EINVAL)):
        assert w(ctypes.byref(desc()), *{**good, **bad}.values()) == rc, bad
    assert w(None, *good.values()) == EINVAL and r(None, *read(good)) == EINVAL


def attention_args(**bad):
    return hip.CachedAttentionArgs(*{**dict(q=A, out=A, page_table=A, kv_len=A, q_start=A, visible=None, work=A, work_bytes=1 << 40, rows=8, ldq=256, ldo=256, seqs=2,
                                            max_pages=4, max_q=4, heads=4, dtype=hip.T_F16, scale=0.1), **bad}.values())


def test_c_attention_refusals():
    f, n = hip.lib().vda_cached_attention, hip.lib().vda_cached_attention_work
    for bad, rc in BAD_CACHES:
        assert f(ctypes.byref(desc(**bad)), ctypes.byref(attention_args()), None) == rc and n(ctypes.byref(desc(**bad)), 2, 4, 4, 4) == rc, bad
    for bad, rc in ((dict(q=None), EINVAL), (dict(out=None), EINVAL), (dict(page_table=None), EINVAL), (dict(kv_len=None), EINVAL), (dict(q_start=None), EINVAL),
                    (dict(rows=0), EINVAL), (dict(seqs=0), EINVAL), (dict(max_pages=0), EINVAL), (dict(max_q=0), EINVAL), (dict(heads=0), EINVAL), (dict(dtype=0), EINVAL),
                    (dict(heads=3), ESHAPE), (dict(ldq=255), ESHAPE), (dict(ldo=248), ESHAPE), (dict(ldq=257), ESHAPE), (dict(q=A + 8), ESHAPE), (dict(out=A + 2), ESHAPE),
                    (dict(max_pages=1 << 27), ESHAPE)):
        assert f(ctypes.byref(desc()), ctypes.byref(attention_args(**bad)), None) == rc, bad
    assert f(ctypes.byref(desc()), None, None) == EINVAL and f(None, ctypes.byref(attention_args()), None) == EINVAL
    for bad, rc in (((0, 4, 4, 4), EINVAL), ((2, 0, 4, 4), EINVAL), ((2, 4, 0, 4), EINVAL), ((2, 4, 4, 0), EINVAL), ((2, 4, 4, 3), ESHAPE), ((2, 1 << 27, 4, 4), ESHAPE)):
        assert n(ctypes.byref(desc()), *bad) == rc, bad


def test_c_attention_refuses_a_missing_or_small_workspace():
    """Sizes whose long axis is split need the workspace."""
    f, n = hip.lib().vda_cached_attention, hip.lib().vda_cached_attention_work
    d = desc(pages=2000, page_size=64)
    need = n(ctypes.byref(d), 1, 1000, 1, 4)
    assert need > 0
    for bad, rc in ((dict(work=None), EINVAL), (dict(work_bytes=need - 1), ESHAPE), (dict(work=A + 4), ESHAPE)):
        assert f(ctypes.byref(d), ctypes.byref(attention_args(seqs=1, max_pages=1000, max_q=1, **bad)), None) == rc, bad


def test_c_norm_refusals():
    f = hip.lib().vda_gated_norm
    good = dict(x=A, b=A, x_out=A, y=A, post_w=A, post_b=A, gate=A, pre_w=A, pre_b=A, mod_scale=A, mod_shift=A, rows=4, ldx=64, ldb=64, ldxo=64, ldy=64, C=64,
                rows_per_group=2, post=1, pre=2, b_type=hip.T_F16, y_type=hip.T_BF16, resid_scale=1.0, eps=1e-6)
    alone = dict(b=None, x_out=None, post=0, post_w=None, post_b=None, gate=None)
    for bad, rc in ((dict(x=None), EINVAL), (dict(rows=0), EINVAL), (dict(C=0), EINVAL), (dict(rows_per_group=0), EINVAL), (dict(post=3), EINVAL), (dict(pre=-1), EINVAL),
                    (dict(b=None), EINVAL), (dict(x_out=None), EINVAL), (dict(alone, y=None), EINVAL), (dict(alone, gate=A), EINVAL), (dict(alone, post=2), EINVAL),
                    (dict(y=None), EINVAL), (dict(y=None, pre=0, mod_scale=None, mod_shift=None, pre_w=None), EINVAL), (dict(b_type=0), EINVAL), (dict(y_type=9), EINVAL),
                    (dict(C=62), ESHAPE), (dict(C=8196, ldx=8196, ldb=8196, ldxo=8196, ldy=8196), ESHAPE), (dict(ldx=60), ESHAPE), (dict(ldb=63), ESHAPE),
                    (dict(ldy=66), ESHAPE), (dict(x=A + 4), ESHAPE), (dict(b=A + 4), ESHAPE), (dict(gate=A + 8), ESHAPE), (dict(ldxo=68), EINVAL), (dict(rows=1 << 50), ESHAPE)):
        assert f(ctypes.byref(hip.GatedNormArgs(*{**good, **bad}.values())), None) == rc, bad
    assert f(None, None) == EINVAL


def test_argument_structs_match_the_header(tmp_path):
    fields = [(n, f) for s, n in ((hip.CacheDesc, "VdaTokenCache"), (hip.CachedAttentionArgs, "VdaCachedAttentionArgs"), (hip.GatedNormArgs, "VdaGatedNormArgs"))
              for f in [x[0] for x in s._fields_]]
    body = "".join('printf("%%zu\\n", offsetof(%s, %s));' % x for x in fields)
    sizes = "".join('printf("%%zu\\n", sizeof(%s));' % n for n in ("VdaTokenCache", "VdaCachedAttentionArgs", "VdaGatedNormArgs"))
    (tmp_path / "t.c").write_text('#include <stdio.h>\n#include <stddef.h>\n#include "vda_hip.h"\nint main(void) {' + body + sizes + "return 0; }\n")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "t.c"), "-o", str(tmp_path / "t")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, check=True).stdout.split()]
    of = {"VdaTokenCache": hip.CacheDesc, "VdaCachedAttentionArgs": hip.CachedAttentionArgs, "VdaGatedNormArgs": hip.GatedNormArgs}
    assert got == [getattr(of[n], f).offset for n, f in fields] + [ctypes.sizeof(s) for s in of.values()]


def test_c_attention_refuses_sizes_beyond_its_counters():
    n = hip.lib().vda_cached_attention_work
    big = (1 << 31) - 1
    for seqs, max_pages, max_q, heads in ((1, 4, big, 4), (big, 4, 1, 4), (big, 4, big, 4), (big, 1 << 20, big, big // 2 * 2), (1, (1 << 30) // 32 + 1, 1, 4)):
        assert n(ctypes.byref(desc()), seqs, max_pages, max_q, heads) == ESHAPE, (seqs, max_pages, max_q, heads)
    assert n(ctypes.byref(desc()), 1, (1 << 30) // 32, 1, 4) > 0


def test_c_cache_refuses_key_heads_that_overflow_a_workgroups_count():
    """32 tokens of 2^27 key heads are 2^32 rows: a 32-bit count of them would be 0 and nothing would be stored."""
    d = desc(pages=1, page_size=16, kv_heads=1 << 27, hd=8)
    row = 8 << 27
    assert hip.lib().vda_cache_write(ctypes.byref(d), A, A, A, 1, row, row, hip.T_F16, None, None, 0, 0, 0, 0, 0, None) == ESHAPE
    assert hip.lib().vda_cache_read(ctypes.byref(d), A, A, A, 1, row, row, hip.T_F16, None) == ESHAPE
    assert hip.lib().vda_cached_attention_work(ctypes.byref(desc(pages=1, page_size=16, kv_heads=65537)), 1, 1, 1, 65537) == ESHAPE


def test_c_attention_in_place_needs_one_stride():
    f = hip.lib().vda_cached_attention
    assert f(ctypes.byref(desc()), ctypes.byref(attention_args(q=A, out=A, ldq=256, ldo=264)), None) == EINVAL


@pytest.fixture
def addressed(monkeypatch):
    """The wrappers with the library replaced by a recorder of the arguments that reach it."""
    calls = []

    class Recorder:
        def __getattr__(self, name):
            return lambda *a: calls.append((name, a)) or 0

    monkeypatch.setattr(hip, "lib", lambda: Recorder())
    monkeypatch.setattr(hip, "_dev", lambda *ts: None)
    monkeypatch.setattr(hip, "_current_device", lambda: -1)
    monkeypatch.setattr(hip, "_stream", lambda: None)
    return calls


ROWS, HEADS, HD = 6, 4, 64
WIDTH = HEADS * HD
# (name, rows of WIDTH values in a tensor whose own strides say where each lies, the stride of a row)
ROW_VIEWS = [("dense", lambda: torch.zeros(ROWS, HEADS, HD), WIDTH), ("flat", lambda: torch.zeros(ROWS * WIDTH), WIDTH), ("frames", lambda: torch.zeros(2, 3, WIDTH), WIDTH),
             ("half rows", lambda: torch.zeros(2 * ROWS, WIDTH // 2), WIDTH), ("columns", lambda: torch.zeros(ROWS, 3 * WIDTH)[:, WIDTH:2 * WIDTH], 3 * WIDTH),
             ("columns of frames", lambda: torch.zeros(2, 3, 3 * WIDTH)[..., WIDTH:2 * WIDTH], 3 * WIDTH), ("part of packed rows", lambda: torch.zeros(ROWS, 3, HEADS, HD)[:, 1], 3 * WIDTH),
             ("wider rows", lambda: torch.zeros(ROWS, 2 * WIDTH), 2 * WIDTH), ("every other row", lambda: torch.zeros(2 * ROWS, WIDTH)[::2], 2 * WIDTH),
             ("a longer buffer", lambda: torch.zeros(ROWS + 2, 2 * WIDTH)[:, :WIDTH], 2 * WIDTH), ("a longer flat one", lambda: torch.zeros(ROWS * WIDTH + 8), WIDTH)]
# the same count of elements behind the first one, but no such rows
NO_ROW_VIEWS = [("one row repeated", lambda: torch.zeros(16, WIDTH)[2:3].expand(ROWS, WIDTH)), ("one row of heads repeated", lambda: torch.zeros(16, HEADS, HD)[2:3].expand(ROWS, HEADS, HD)),
                ("heads apart", lambda: torch.zeros(ROWS * HEADS, 2 * HD)[:, :HD]), ("overlapping windows", lambda: torch.zeros(16 * WIDTH).as_strided((ROWS, WIDTH), (64, 1))),
                ("frames apart", lambda: torch.zeros(8, 4, WIDTH)[:2, 1:]), ("rows of frames, more of them", lambda: torch.zeros(8, 4, WIDTH)),
                ("a strided line", lambda: torch.zeros(4 * ROWS * WIDTH)[::2]), ("packed rows taken for rows", lambda: torch.zeros(ROWS + 1, 3, WIDTH)),
                ("turned", lambda: torch.zeros(16 * WIDTH, 16).t()[:ROWS, :WIDTH]), ("a shorter view of a longer buffer", lambda: torch.zeros(16, WIDTH)[:ROWS - 1]),
                ("a shorter line of a longer buffer", lambda: torch.zeros(16 * WIDTH)[:ROWS * WIDTH - 1])]


def row_calls(addressed):
    """For each wrapper and each of its row operands: a call with that operand given, and where its stride is found."""
    f = f16
    pos, freq, slots = torch.zeros(ROWS, 3, dtype=i32), torch.zeros(32, dtype=f64), torch.zeros(ROWS, dtype=i64)
    p = planes(heads=HEADS, hd=HD)
    seq = torch.zeros(1, 3, dtype=i32), torch.zeros(1, dtype=i32), torch.zeros(2, dtype=i32)
    good = lambda t=f: torch.zeros(ROWS, WIDTH, dtype=t)  # noqa: E731
    rot, cache = dict(rows=ROWS, heads=HEADS, hd=HD, sections=(8, 12, 12)), dict(rows=ROWS, kv_heads=HEADS, hd=HD, page_size=16, fmt=hip.CACHE_I8)
    att = dict(heads=HEADS, kv_heads=HEADS, hd=HD, page_size=16, fmt=hip.CACHE_I8, max_q=ROWS, scale=0.1, rows=ROWS)
    norm = lambda x=None, b=None, x_out=None, y=None: hip.gated_norm(good(f32) if x is None else x, good() if b is None else b, good(f32) if x_out is None else x_out,  # noqa: E731
                                                                     good() if y is None else y, rows=ROWS, C=WIDTH)
    arg = lambda i: lambda: addressed[-1][1][i]  # noqa: E731
    field = lambda name, which: lambda: getattr(which.from_buffer_copy(addressed[-1][1][1 if which is hip.CachedAttentionArgs else 0]), name)  # noqa: E731
    return [(f, lambda t: hip.rotary_axes(t, good(), pos, freq, **rot), arg(7)), (f, lambda t: hip.rotary_axes(good(), t, pos, freq, **rot), arg(8)),
            (f, lambda t: hip.cache_write(t, good(), *p, slots, **cache), arg(5)), (f, lambda t: hip.cache_write(good(), t, *p, slots, **cache), arg(6)),
            (f, lambda t: hip.cache_read(*p, slots, t, good(), **cache), arg(5)), (f, lambda t: hip.cache_read(*p, slots, good(), t, **cache), arg(6)),
            (f, lambda t: hip.cached_attention(t, good(), *p, *seq, **att), field("ldq", hip.CachedAttentionArgs)),
            (f, lambda t: hip.cached_attention(good(), t, *p, *seq, **att), field("ldo", hip.CachedAttentionArgs)),
            (f32, lambda t: norm(x=t), field("ldx", hip.GatedNormArgs)), (f, lambda t: norm(b=t), field("ldb", hip.GatedNormArgs)),
            (f32, lambda t: norm(x_out=t), field("ldxo", hip.GatedNormArgs)), (f, lambda t: norm(y=t), field("ldy", hip.GatedNormArgs))]


@pytest.mark.parametrize("name,make,ld", ROW_VIEWS, ids=[v[0] for v in ROW_VIEWS])
def test_rows_lie_where_the_tensors_strides_say(addressed, name, make, ld):
    for dtype, call, stride in row_calls(addressed):
        call(make().to(dtype) if make().is_contiguous() else torch.zeros(make().untyped_storage().nbytes() // 4, dtype=dtype).as_strided(make().shape, make().stride(), make().storage_offset()))
        assert stride() == ld


@pytest.mark.parametrize("name,make", NO_ROW_VIEWS, ids=[v[0] for v in NO_ROW_VIEWS])
def test_tensors_whose_strides_make_no_such_rows_are_refused(addressed, name, make):
    """Their memory reaches far enough: taken for dense rows, the call would read and write values of other rows or none."""
    for dtype, call, _ in row_calls(addressed):
        t = make()
        t = torch.zeros(t.untyped_storage().nbytes() // 4, dtype=dtype).as_strided(t.shape, t.stride(), t.storage_offset())
        with pytest.raises(ValueError):
            call(t)


def test_a_row_stride_that_is_given_counts_from_the_tensors_first_element(addressed):
    pos, freq = torch.zeros(ROWS, 3, dtype=i32), torch.zeros(32, dtype=f64)
    kw = dict(rows=ROWS, heads=HEADS, hd=HD, sections=(8, 12, 12))
    out, buf = torch.zeros(ROWS, WIDTH, dtype=f16), torch.zeros(ROWS * 3 * WIDTH, dtype=f16)
    for t in (buf, buf[WIDTH:], buf.view(ROWS, 3, HEADS, HD)[:, 1], buf.view(1, ROWS, 3 * WIDTH)[..., :WIDTH]):
        hip.rotary_axes(t, out, pos, freq, ldx=3 * WIDTH, **kw)
        assert addressed[-1][1][7] == 3 * WIDTH
    for bad in (buf[2 * WIDTH + 8:], torch.zeros(8 * ROWS, 2 * HD, dtype=f16)[:, :HD]):          # beyond the memory; a row that is not dense
        with pytest.raises(ValueError):
            hip.rotary_axes(bad, out, pos, freq, ldx=3 * WIDTH, **kw)


def test_vectors_and_workspaces_end_where_the_tensor_does(addressed, monkeypatch):
    """A tensor that is shorter than the call needs is refused, also where the memory behind it goes on: what lies there is another
    tensor's (the next frame's gate, another call's workspace)."""
    whole = lambda dtype: torch.zeros(64, WIDTH, dtype=dtype)  # noqa: E731
    x, y, b = torch.zeros(ROWS, WIDTH), torch.zeros(ROWS, WIDTH, dtype=f16), torch.zeros(ROWS, WIDTH, dtype=f16)
    norm = dict(rows=ROWS, C=WIDTH, rows_per_group=2)
    gates, w = whole(f32)[:3], whole(f32)[0]
    hip.gated_norm(x, b, x, y, gate=gates, mod_scale=gates, mod_shift=gates, post_w=w, post_b=w, pre_w=w, pre_b=w, **norm)
    for name, t in (("gate", whole(f32)[0]), ("mod_scale", whole(f32)[:2]), ("mod_shift", whole(f32)[:2]), ("post_w", whole(f32)[0, :-1]), ("post_b", whole(f32)[0, :-1]),
                    ("pre_w", whole(f32)[0, 1:]), ("pre_b", whole(f32)[0, 1:])):
        with pytest.raises(ValueError, match=f"{name} holds"):
            hip.gated_norm(x, b, x, y, **{name: t}, **norm)
    pos, freq, slots = torch.zeros(64, 3, dtype=i32), torch.zeros(64, dtype=f64), torch.zeros(64, dtype=i64)
    rot = dict(rows=ROWS, heads=HEADS, hd=HD, sections=(8, 12, 12))
    hip.rotary_axes(b, y, pos[:ROWS], freq[:32], **rot)
    for p, f, name in ((pos[:ROWS - 1], freq, "pos"), (pos, freq[:31], "freq")):
        with pytest.raises(ValueError, match=f"{name} holds"):
            hip.rotary_axes(b, y, p, f, **rot)
    p = planes(heads=HEADS, hd=HD)
    cache = dict(kv_heads=HEADS, hd=HD, page_size=16, fmt=hip.CACHE_I8)
    for call in (lambda: hip.cache_write(b, y, *p, slots[:ROWS - 1], rows=ROWS, **cache), lambda: hip.cache_read(*p, slots[:ROWS - 1], b, y, rows=ROWS, **cache)):
        with pytest.raises(ValueError, match="slots holds"):
            call()
    seq = torch.zeros(1, 3, dtype=i32), torch.zeros(1, dtype=i32), torch.zeros(2, dtype=i32)
    att = dict(heads=HEADS, max_q=ROWS, scale=0.1, **cache)
    with pytest.raises(ValueError, match="visible holds"):
        hip.cached_attention(b, y, *p, *seq, visible=torch.zeros(64, dtype=i32)[:ROWS - 1], **att)

    class Needs:
        vda_cached_attention_work = staticmethod(lambda *a: 4096)
        vda_cached_attention = staticmethod(lambda *a: 0)

    monkeypatch.setattr(hip, "lib", lambda: Needs)
    arena = torch.zeros(4 * 4096, dtype=u8)
    hip.cached_attention(b, y, *p, *seq, work=arena[4096:8192], **att)
    hip.cached_attention(b, y, *p, *seq, work=arena.view(f32)[:1024], **att)
    for work in (arena[4096:8191], arena.view(f32)[:1023], arena[::2][:4096]):
        with pytest.raises(ValueError, match="work"):
            hip.cached_attention(b, y, *p, *seq, work=work, **att)


def test_attention_kernels_do_not_promise_that_queries_and_outputs_lie_apart():
    """`out` may be `q`: a __restrict__ on either would let the compiler read q after it has written out."""
    import re
    csrc = os.path.join(ROOT, "monocular-depth-estimation_amd", "csrc")
    for name in ("cached_attention_few.hip", "cached_attention_many.hip"):
        heads = re.findall(r"void\s+(attend_(?:few|many)_kernel)\(([^)]*)\)", open(os.path.join(csrc, name)).read())
        assert len(heads) == 1
        assert "__restrict__" not in heads[0][1], heads


def test_c_attention_refuses_a_scale_that_is_no_number():
    """One kernel would take it for 0, the other give NaN."""
    f = hip.lib().vda_cached_attention
    for scale in (float("nan"), float("inf"), -float("inf"), 3e38):
        assert f(ctypes.byref(desc()), ctypes.byref(attention_args(scale=scale)), None) == EINVAL, scale
