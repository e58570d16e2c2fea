"""Plain 64-bit statements of the operators for video transformers with a token memory, on the CPU, and the bounds their kernels are
held to.  A rounding to a type is off by at most half a step, eps / 2 of the value."""
import math

import torch

LARGEST = {"i8": 127.0, "e4m3": 448.0}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rotate(x, pos, freq, sections, pairing):
    """(turned rows, |a| + |b| of every channel's pair) in float64; x [rows, heads, hd]."""
    x, freq = x.double().cpu(), freq.double().cpu()
    n = freq.numel()
    axis = torch.tensor([0] * sections[0] + [1] * sections[1] + [2] * sections[2])
    angle = pos.double().cpu()[:, axis] * freq
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    i = torch.arange(n) if pairing == "halves" else torch.arange(0, 2 * n, 2)
    j = i + (n if pairing == "halves" else 1)
    y, size = x.clone(), x.abs()
    y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
    size[..., i] = size[..., j] = x[..., i].abs() + x[..., j].abs()
    return y, size


# The rotation in fp32: the angle's remainder is rounded once (half a turn in 24 bits: 1e-7 rad), cosine and sine are good to 2 ulp
# (2.4e-7), two products and their sum round (1.8e-7), each relative to |a| + |b|.
ROTATION = 6e-7


def exponents(x, fmt):
    """The exponent bytes of the rows of x (last axis), from the rule: the smallest e in 1 .. 254 with max|x| <= largest * 2^(e - 127)."""
    amax = x.double().abs().amax(-1)
    e = torch.full(amax.shape, 1, dtype=torch.int64)
    for k in range(2, 255):                        # as often as a row's magnitude exceeds what exponent k - 1 holds
        e[amax > LARGEST[fmt] * 2.0 ** (k - 1 - 127)] = k
    e[~torch.isfinite(amax)] = 255
    return e


def codes(x, e, fmt):
    """The values that the codes stand for before scaling, float64."""
    y = x.double() * torch.exp2(127.0 - e.double())[..., None]
    return torch.round(y) if fmt == "i8" else y.float().to(torch.float8_e4m3fn).double()


def decode(plane, exps, fmt):
    c = plane.cpu().contiguous().view(torch.int8 if fmt == "i8" else torch.float8_e4m3fn).double()
    v = c * torch.exp2(exps.cpu().double() - 127.0)[..., None]
    return torch.where((exps.cpu() == 255)[..., None], torch.full((), math.nan, dtype=torch.float64), v)


def attend(q, ck, cv, ek, ev, table, kv_len, q_start, visible, heads, kv_heads, hd, page, fmt, scale):
    """(output, bound of the kernel's error) in float64, one row and head at a time in the order of the definition; rows of no
    sequence are NaN.  The bound counts: probabilities rounded to 11 bits (16-bit q) or two pieces of 22 (fp32 q), scores off by the
    fp32 sum of hd products, sums over n keys whose roundings are independent, the rounding of the result."""
    q, table, kv_len, q_start = q.cpu(), table.cpu(), kv_len.cpu().tolist(), q_start.cpu().tolist()
    fp32 = q.dtype == torch.float32
    out = torch.full((q.shape[0], heads, hd), math.nan, dtype=torch.float64)
    tol = torch.zeros_like(out)
    k_all, v_all, e_all = decode(ck, ek, fmt)[..., :hd], decode(cv, ev, fmt)[..., :hd], ek.cpu()
    G, pages = heads // kv_heads, ck.shape[0]
    for s in range(len(kv_len)):
        n = max(0, min(kv_len[s], table.shape[1] * page))
        held = -(-n // page)
        t = table[s, :held].long()
        there = (t >= 0) & (t < pages)
        t = torch.where(there, t, torch.zeros_like(t))
        take = lambda a: a[t].transpose(0, 1).flatten(1, 2)[:, :n]  # noqa: E731
        k, v = take(k_all), take(v_all)                              # [kv_heads, n, hd]
        seen = take(e_all).ne(0) & there.repeat_interleave(page)[:n]
        for r in range(max(0, q_start[s]), min(q.shape[0], q_start[s + 1])):
            limit = n if visible is None else max(0, min(n, int(visible[r])))
            for h in range(heads):
                look = seen[h // G].clone()
                look[limit:] = False
                kk, vv = k[h // G][look], v[h // G][look]
                if kk.shape[0] == 0:
                    out[r, h] = 0.0
                    continue
                qq = q[r].double().reshape(heads, hd)[h]
                sc = (kk @ qq) * scale
                w = torch.softmax(sc, 0)
                o, size = w @ vv, w @ vv.abs()
                m = kk.shape[0]
                sums = 4 * (8 + math.sqrt(m)) * 2.0 ** -24
                dots = 2 * (hd + 8) * 2.0 ** -24 * float(((kk.abs() @ qq.abs()) * abs(scale)).max())
                pieces = 2.0 ** -20 if fp32 else 2.0 ** -11
                e = size * (pieces + sums + dots)
                out[r, h], tol[r, h] = o, e + half_step(q.dtype) * (o.abs() + e)
    return out, tol


def norm(x, kind, eps):
    if kind == "none":
        return x
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)


def gated_norm(x, b, post, post_w, post_b, gate, resid_scale, pre, pre_w, pre_b, mod_scale, mod_shift, per, eps):
    """(x_out, y, sizes of the terms they are sums of) in float64."""
    d = lambda t: None if t is None else t.double().cpu()  # noqa: E731
    x, b = d(x), d(b)
    g = torch.arange(x.shape[0]) // per
    size_x = x.abs()
    if b is not None:
        n = norm(b, post, eps)
        size = n.abs() + (b.abs().mean(-1, keepdim=True) * (n.abs().amax(-1, keepdim=True) / b.abs().amax(-1, keepdim=True).clamp_min(1e-300)) if post == "layer" else 0.0)
        for t, mul in ((post_w, True), (post_b, False)):
            if t is not None:
                n, size = (n * d(t), size * d(t).abs()) if mul else (n + d(t), size + d(t).abs())
        if gate is not None:
            n, size = n * d(gate)[g], size * d(gate)[g].abs()
        x, size_x = resid_scale * x + n, abs(resid_scale) * size_x + size
    y = norm(x, pre, eps)
    rstd = torch.ones(())
    if pre != "none":
        z = x - x.mean(-1, keepdim=True) if pre == "layer" else x
        rstd = 1 / torch.sqrt((z * z).mean(-1, keepdim=True) + eps)
    size_y = (size_x + (x.abs().mean(-1, keepdim=True) + size_x.mean(-1, keepdim=True))) * rstd + y.abs()
    for t, s in ((pre_w, pre_b), (None if mod_scale is None else 1 + d(mod_scale)[g], None if mod_shift is None else d(mod_shift)[g])):
        if t is not None:
            y, size_y = y * d(t), size_y * d(t).abs()
        if s is not None:
            y, size_y = y + d(s), size_y + d(s).abs()
    return x, y, size_x, size_y
