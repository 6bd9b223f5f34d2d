"""tsn_rope_axes, tsn_gate_add_norm and tsn_diff_attention against their formulas in 64 bits, at the sizes, types,
strides and masks where they can go wrong, and one run of them together.

Tolerances follow from the arithmetic, with u = 2^-24 (f32), 2^-11 (f16), 2^-8 (bf16) for one rounding, e = 2^-24:
they are bounds on every element, from the magnitudes of the terms that a result is made of."""
import numpy as np
import pytest

from conftest import rel_l2, rng

pytestmark = pytest.mark.gpu

F32, F16, BF16 = 0, 1, 2
U = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F32: 2.0 ** -126, F16: 2.0 ** -25, BF16: 2.0 ** -126}   # below the normal range: half a subnormal step and less
E = 2.0 ** -24
SENTINEL = {F32: np.float32(-7.0), F16: np.float16(-7.0), BF16: np.uint16(0xC0E0)}
NP = {F32: np.float32, F16: np.float16, BF16: np.uint16}


def enc(a, dt):
    """f32 values rounded to dt, as the device array's elements (bf16: bits, nearest even; NaN stays NaN)"""
    a = np.asarray(a, np.float32)
    if dt != BF16:
        return a.astype(NP[dt])
    b = a.view(np.uint32).astype(np.uint64)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(a), np.uint16(0x7FC0), r)


def dec(a, dt):
    return ((a.astype(np.uint32) << 16).view(np.float32) if dt == BF16 else a).astype(np.float64)


def strided(rows, ld, dt, col=0, fill=None):
    """[n][ld] elements holding rows [n][w] from column col on, `fill` (the sentinel) elsewhere"""
    n, w = rows.shape
    a = np.full((n, ld), SENTINEL[dt] if fill is None else fill, NP[dt])
    a[:, col:col + w] = rows
    return a


class At:
    """a device address inside an array"""

    def __init__(self, arr, elems):
        self.p, self.nbytes = arr.offset(elems), arr.nbytes - elems * arr.dtype.itemsize


def check(got, want, tol, what=""):
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), "%s: %d of %d, first %s: got %r want %r tol %r" % (
        what, bad.sum(), bad.size, np.argwhere(bad)[0], got[bad][0], want[bad][0], np.broadcast_to(tol, got.shape)[bad][0])


# ---------------------------------------------------------------- rotary positions

def rope_ref(x, pos, dims, bases, fscales, half, inverse):
    """x [rows][nh][hd] in f64, pos [rows][axes]"""
    y, at = x.copy(), 0
    for a, d in enumerate(dims):
        i = np.arange(d // 2)
        ang = pos[:, a, None].astype(np.float64) * (np.float64(np.float32(fscales[a])) * np.float64(np.float32(bases[a])) ** (-2.0 * i / max(d, 1)))
        cs, sn = np.cos(ang)[:, None], np.sin(ang)[:, None] * (-1.0 if inverse else 1.0)
        e0, e1 = (at + i, at + i + d // 2) if half else (at + 2 * i, at + 2 * i + 1)
        y[..., e0], y[..., e1] = x[..., e0] * cs - x[..., e1] * sn, x[..., e0] * sn + x[..., e1] * cs
        at += d
    return y


def rope_tol(x, dt, want, dims, half):
    # the reduced angle is rounded once (half a turn: 2^-26 turns, 2^-23.3 rad), sine and cosine are within 4 units of
    # their last place (2^-22 absolute), products and sum 3 roundings: 2^-23.3 + 2^-22 + 3*2^-24 < 2^-20 of |x0| + |x1|;
    # then one rounding to the type
    m, at = np.zeros_like(x), 0
    for d in dims:
        i = np.arange(d // 2)
        e0, e1 = (at + i, at + i + d // 2) if half else (at + 2 * i, at + 2 * i + 1)
        s = np.abs(x[..., e0]) + np.abs(x[..., e1])
        m[..., e0], m[..., e1] = s, s
        at += d
    t = 2.0 ** -20 * m
    return np.where(m > 0, t + U[dt] * (np.abs(want) + t) + TINY[dt], 0.0)   # what no axis turns is copied


ROPES = [
    # dtype rows nh hd dims half inverse ldx ldy col pos_rows
    (F32, 1, 1, 2, (2,), False, False, 0, 0, 0, 0),
    (F32, 2, 32, 64, (16, 24, 24), False, False, 0, 0, 0, 1),
    (F16, 65, 16, 64, (16, 24, 24), False, False, 0, 0, 0, 0),
    (BF16, 130, 8, 64, (32, 16), True, False, 0, 0, 0, 65),
    (F16, 37, 5, 128, (32, 32, 48), True, False, 0, 0, 0, 0),        # a copied tail
    (BF16, 37, 5, 128, (32, 32, 48), True, True, 1024, 800, 64, 0),
    (F32, 33, 3, 80, (8, 24, 16), True, False, 0, 0, 0, 11),
    (F16, 41, 3, 80, (8, 24, 16), False, True, 0, 0, 0, 0),
    (F16, 17, 3, 80, (12, 28, 20), True, False, 0, 0, 0, 0),         # halves that are no multiple of 8
    (F16, 65, 16, 64, (16, 24, 24), True, False, 0, 0, 0, 13),       # halves of 12: chunks of 8 bytes
    (BF16, 37, 5, 60, (24, 24), True, True, 308, 0, 4, 0),           # rows aligned to 8 bytes
    (F16, 1000, 3, 200, (40, 56, 72), True, False, 0, 604, 0, 0),
    (BF16, 37, 5, 60, (24, 24), True, True, 310, 0, 2, 0),           # and to 4
    (F32, 65, 6, 80, (4, 12, 20), True, False, 0, 504, 0, 13),       # halves of 2, 6 and 10
    (F16, 300, 20, 128, (4, 28, 60), True, False, 0, 0, 0, 100),
    (BF16, 37, 5, 58, (4, 24), True, True, 299, 0, 3, 0),            # one element at a time
    (F16, 29, 7, 64, (16, 24, 24), False, False, 1344, 0, 448, 0),   # k heads out of q|k|v rows
    (F16, 29, 7, 64, (16, 24, 24), False, False, 451, 449, 1, 0),    # odd strides
    (BF16, 19, 3, 70, (10, 20, 30, 4), False, False, 0, 0, 0, 0),    # a width that is no multiple of 8, four axes
    (F32, 19, 3, 70, (10, 20, 30, 10), True, False, 0, 0, 0, 0),
    (F32, 50, 4, 256, (64, 96, 96), True, False, 0, 0, 0, 0),
    (BF16, 50, 4, 256, (256,), False, False, 0, 0, 0, 0),
    (F16, 9, 2, 32, (0, 16, 0, 8), False, False, 0, 0, 0, 0),        # empty axes
    (F16, 9, 2, 64, (0,), True, False, 0, 0, 0, 0),                  # nothing turns
    (BF16, 1000, 40, 64, (16, 24, 24), False, False, 0, 0, 0, 500),
    (F32, 3, 1, 8, (8,), True, False, 0, 0, 0, 0),
    (F16, 700, 1, 8, (8,), False, False, 0, 0, 0, 7),
    (BF16, 300, 3, 16, (16,), True, False, 0, 0, 0, 0),
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("dt,rows,nh,hd,dims,half,inverse,ldx,ldy,col,pos_rows", ROPES)
def test_rope_axes(tsn, rt, dt, rows, nh, hd, dims, half, inverse, ldx, ldy, col, pos_rows, in_place):
    r = rng(rows * 131 + hd)
    n, k = nh * hd, len(dims)
    x = enc(r.standard_normal((rows, n)), dt)
    pr = pos_rows or rows
    pos = r.integers(-50, 4000, (pr, k)).astype(np.int32)
    if pr > 2:   # far positions: 32-bit angles would be off by whole radians
        pos[1], pos[2] = 2 ** 31 - 1, -2 ** 31
    bases, fs = (10000.0, 100.0, 50.0, 7.5)[:k], (1.0, 2.6875, 0.5, 1.0)[:k]
    ldx = ldx or n
    ldy = ldx if in_place else (ldy or n)
    xb = rt.array(strided(x, ldx, dt, col if ldx > n else 0))
    c = col if ldx > n else 0
    yb = xb if in_place else rt.array(np.full((rows, ldy), SENTINEL[dt], NP[dt]))
    spec = tsn.rope_axes_spec(dt, rows, nh, hd, dims, bases, fs, ldx=ldx, ldy=ldy, pos_rows=pos_rows, half_split=half, inverse=inverse)
    posb = rt.array(pos)
    rt.rope_axes(spec, At(xb, c), posb, At(yb, c if in_place else 0))
    rt.sync()
    out = yb.numpy()
    cy = c if in_place else 0
    got = dec(out[:, cy:cy + n], dt).reshape(rows, nh, hd)
    xf = dec(x, dt).reshape(rows, nh, hd)
    want = rope_ref(xf, pos[np.arange(rows) % pr], dims, bases, fs, half, inverse)
    check(got, want, rope_tol(xf, dt, want, dims, half))
    rest = np.delete(out, np.s_[cy:cy + n], 1)
    assert (rest == SENTINEL[dt]).all()   # columns outside the heads are left as they were
    for b in {id(xb): xb, id(yb): yb, id(posb): posb}.values():
        b.free()


def spread(n, r):
    """rows of a large array that are looked at: both ends and some between"""
    return np.unique(np.concatenate([np.arange(40), r.integers(0, n, 400), np.arange(n - 40, n)]))


@pytest.mark.parametrize("dt,half,dims", [(F32, False, (16, 16, 32)), (F16, True, (16, 16, 32)), (F16, False, (16, 16, 32)),
                                          (BF16, True, (16, 16, 32)), (F16, True, (16, 24, 24))])
def test_rope_axes_large(tsn, rt, dt, half, dims):
    """traffic past the last-level cache (over 192 MiB), an odd number of rows"""
    r = rng(12)
    nh, hd, bases = 32, 64, (1e4, 1e2, 1e2)
    rows = (13 if dt == F32 else 26) * 1000 + 1
    some = enc(r.standard_normal((997, nh * hd)), dt)
    x = some[np.arange(rows) % 997]
    pos = r.integers(0, 5000, (rows, 3)).astype(np.int32)
    xb, pb, yb = rt.array(x), rt.array(pos), rt.array(np.full(x.shape, SENTINEL[dt], NP[dt]))
    rt.rope_axes(tsn.rope_axes_spec(dt, rows, nh, hd, dims, bases, half_split=half), xb, pb, yb)
    rt.sync()
    at = spread(rows, r)
    got, xf = dec(yb.numpy()[at], dt).reshape(len(at), nh, hd), dec(x[at], dt).reshape(len(at), nh, hd)
    want = rope_ref(xf, pos[at], dims, bases, (1.0,) * 3, half, False)
    check(got, want, rope_tol(xf, dt, want, dims, half))
    for b in (xb, pb, yb):
        b.free()


def test_rope_axes_one_axis_is_rope_pairs(tsn, rt):
    """n_axes = 1 over the whole head is tsn_rope_pairs; its angle is rounded to f32 at up to 171 rad (2^-17 of a
    radian), its product with the frequency and powf add as much again twice: 2^-15 of |x0| + |x1| between the two"""
    r = rng(5)
    rows, nh, hd = 172, 16, 64
    x = r.standard_normal((rows, nh * hd)).astype(np.float32)
    a, pos = rt.array(x), rt.array(np.arange(rows, dtype=np.int32))
    y = rt.empty(x.shape)
    rt.rope_axes(tsn.rope_axes_spec(F32, rows, nh, hd, (hd,), (10000.0,)), a, pos, y)
    rt.rope_pairs(a, pos, rows, nh, nh * hd, hd, 0, 0, 1.0, 10000.0)
    rt.sync()
    m = np.abs(x.reshape(rows, -1, 2)).sum(-1).repeat(2, -1)
    check(y.numpy().astype(np.float64), a.numpy().astype(np.float64), 2.0 ** -15 * m)


def test_rope_axes_turns_back(tsn, rt):
    """inverse undoes the turn within two roundings to f32 and two evaluations"""
    r = rng(6)
    rows, nh, hd, dims, bases = 77, 6, 64, (16, 24, 24), (1e4, 1e2, 1e2)
    x = r.standard_normal((rows, nh * hd)).astype(np.float32)
    a, pos = rt.array(x), rt.array(r.integers(0, 100000, (rows, 3)).astype(np.int32))
    for inv in (False, True):
        rt.rope_axes(tsn.rope_axes_spec(F32, rows, nh, hd, dims, bases, inverse=inv), a, pos, a)
    rt.sync()
    m = np.abs(x.reshape(rows, -1, 2)).sum(-1).repeat(2, -1)
    check(a.numpy().astype(np.float64), x.astype(np.float64), 2 * 2.0 ** -20 * m * np.sqrt(2.0))


# ---------------------------------------------------------------- norms around a block

def norm_ref(kind, x, w, b, eps, ex):
    """(norm, bound) of x [rows][H] known to ex; sums of H squares by a tree over threads that each add at most
    H/64 terms: relative error D"""
    H = x.shape[1]
    D = E * (H / 64 + 16)
    if kind == 0:
        y, t = x, ex
    else:
        mean = x.mean(-1, keepdims=True) if kind == 2 else 0.0
        d = x - mean
        em = (ex + D * np.abs(x)).mean(-1, keepdims=True) if kind == 2 else 0.0   # of the mean
        ed = ex + em + E * np.abs(d)
        ms = (d * d).mean(-1, keepdims=True) + eps
        inv = 1.0 / np.sqrt(ms)
        # relative error of inv: half that of the mean square (its terms' and the sum's), and three roundings
        ei = 0.5 * ((2 * np.abs(d) * ed + ed * ed).mean(-1, keepdims=True) / ms + D) + 4 * E
        y, t = d * inv, ed * inv * (1 + ei) + np.abs(d) * inv * (ei + 2 * E)
    if w is not None:
        y, t = y * w, t * np.abs(w) + E * np.abs(y * w)
    if b is not None:
        y, t = y + b, t + E * (np.abs(y) + np.abs(b))
    return y, t


def gate_norm_ref(x, f, mod, c, ws):
    """(x_out, bound, y, bound) before the roundings to the outputs' types"""
    rows, H = x.shape
    z, tz = norm_ref(c["post"], f, ws.get("post_w"), ws.get("post_b"), c["post_eps"], np.zeros_like(f))
    chunk = lambda i: mod[np.arange(rows) // c["mod_rows"], i * H:(i + 1) * H]  # noqa: E731
    g = np.float64(np.float32(c["f_scale"])) * (chunk(c["gate"]) if c["gate"] >= 0 else 1.0)
    xs = np.float64(np.float32(c["x_scale"])) * x
    xo = xs + g * z
    ex = np.abs(g) * tz + 4 * E * (np.abs(xs) + np.abs(g * z))
    y, ty = norm_ref(c["pre"], xo, ws.get("pre_w"), ws.get("pre_b"), c["pre_eps"], ex)
    if c["scale"] >= 0:
        s = 1.0 + chunk(c["scale"])
        y, ty = y * s, ty * np.abs(s) + 3 * E * (np.abs(y) * (1 + np.abs(s - 1)))
    if c["shift"] >= 0:
        sh = chunk(c["shift"])
        y, ty = y + sh, ty + 2 * E * (np.abs(y) + np.abs(sh))
    return xo, ex, y, ty


NORMS = [
    # rows H xdt fdt ydt post pre mod_rows chunks(gate, shift, scale) weights ld(x, f, o, y)
    (1, 1, F32, F32, F32, 1, 2, 1, (2, 0, 1), True, None),
    (1, 64, F32, F16, BF16, 2, 1, 1, (2, 0, 1), False, None),
    (8, 1024, F32, F32, F32, 1, 1, 4, (2, 0, 1), True, None),
    (397, 1024, F32, F16, F16, 1, 2, 397, (5, 3, 4), True, None),
    (33, 1024, BF16, BF16, BF16, 2, 2, 1, (0, 1, 2), True, None),
    (5, 1023, F32, F16, F16, 2, 1, 2, (2, 0, 1), True, None),              # odd width
    (7, 1025, BF16, F32, F16, 1, 2, 3, (2, 0, 1), True, None),
    (6, 520, F16, BF16, F32, 1, 1, 4, (2, 0, 1), False, (520, 528, 536, 544)),
    (6, 520, F16, BF16, F32, 1, 1, 4, (2, 0, 1), True, (521, 523, 525, 527)),   # odd strides
    (9, 2048, F16, F16, F16, 2, 0, 9, (-1, 0, 1), False, None),
    (9, 2816, F32, F32, F16, 0, 1, 2, (1, -1, 0), True, None),
    (4, 4096, BF16, F16, F32, 1, 2, 1, (2, 0, 1), True, None),
    (3, 8192, F32, BF16, F16, 2, 1, 1, (-1, -1, -1), True, None),
    (3, 16384, F32, F32, F32, 2, 2, 2, (2, 0, 1), True, None),
    (2, 12345, F16, F32, BF16, 1, 2, 1, (2, 0, 1), False, None),
    (3, 16, F32, F32, F32, 0, 0, 1, (2, 0, 1), False, None),
    (1003, 264, BF16, BF16, F32, 1, 1, 100, (2, 0, 1), True, None),
    (515, 72, F32, F16, F16, 2, 2, 5, (2, 0, 1), False, None),
    (77, 333, F16, F32, BF16, 2, 2, 7, (2, 0, 1), True, None),             # one by one: one wave, four, eight
    (19, 1777, BF16, F16, F32, 1, 2, 3, (2, 0, 1), True, (1777, 1779, 1781, 1783)),
    (19, 2501, BF16, BF16, BF16, 2, 1, 1, (2, 0, 1), False, None),
    (5, 4095, F32, F32, F32, 2, 2, 2, (2, 0, 1), True, None),
    (5, 4097, F32, F16, F32, 1, 1, 2, (2, 0, 1), True, None),              # sixteen
    (7, 8191, BF16, F32, F16, 2, 2, 3, (2, 0, 1), True, None),
    (5, 8193, F32, F16, F32, 1, 1, 2, (2, 0, 1), True, None),              # past what registers hold
    (5, 3328, F32, F16, F32, 1, 1, 2, (2, 0, 1), True, None),              # whole chunks, eight waves
]


@pytest.mark.parametrize("mode", ["apart", "in_place", "no_y"])
@pytest.mark.parametrize("rows,H,xdt,fdt,ydt,post,pre,mod_rows,chunks,weights,lds", NORMS)
def test_gate_add_norm(tsn, rt, rows, H, xdt, fdt, ydt, post, pre, mod_rows, chunks, weights, lds, mode):
    r = rng(rows * 7 + H)
    ldx, ldf, ldo, ldy = lds or (H,) * 4
    if mode == "in_place":
        ydt, ldo, ldy = fdt, ldx, ldf
    x, f = enc(3.0 * r.standard_normal((rows, H)) + 0.5, xdt), enc(0.7 * r.standard_normal((rows, H)) - 0.2, fdt)
    if rows > 2:
        f[1] = enc(np.full(H, 0.0), fdt)         # a row of zeros: eps alone
        x[2] = enc(np.full(H, 100.0), xdt)       # a row far from zero
    nch = max(chunks) + 1
    mod = (0.3 * r.standard_normal((-(-rows // mod_rows), nch * H))).astype(np.float32) if nch else None
    ws = {n: (1.0 * n.endswith("w") + 0.1 * r.standard_normal(H)).astype(np.float32)
          for n in ("post_w", "post_b", "pre_w", "pre_b")} if weights else {}
    c = dict(post=post, pre=pre, x_scale=0.9, f_scale=1.1, mod_rows=mod_rows, gate=chunks[0], shift=chunks[1], scale=chunks[2],
             post_eps=1e-5, pre_eps=1e-6)
    spec = tsn.gate_norm_spec(rows, H, xdt, fdt, ydt, chunks=nch, ldx=ldx, ldf=ldf, ldo=ldo, ldy=ldy, **c)
    xb, fb = rt.array(strided(x, ldx, xdt)), rt.array(strided(f, ldf, fdt))
    mb = rt.array(mod) if nch else None
    wb = {n: rt.array(w) for n, w in ws.items()}
    ob = xb if mode == "in_place" else rt.array(np.full((rows, ldo), SENTINEL[xdt], NP[xdt]))
    yb = None if mode == "no_y" else fb if mode == "in_place" else rt.array(np.full((rows, ldy), SENTINEL[ydt], NP[ydt]))
    rt.gate_add_norm(spec, xb, fb, mb, ob, yb, **wb)
    rt.sync()
    c["post_eps"], c["pre_eps"] = (np.float64(np.float32(c[k])) for k in ("post_eps", "pre_eps"))
    xo, ex, y, ty = gate_norm_ref(dec(x, xdt), dec(f, fdt), mod, c, {n: w.astype(np.float64) for n, w in ws.items()})
    got = ob.numpy()
    check(dec(got[:, :H], xdt), xo, ex + U[xdt] * (np.abs(xo) + ex) + TINY[xdt], "x_out")
    assert (got[:, H:] == SENTINEL[xdt]).all()
    if yb is not None:
        got = yb.numpy()
        check(dec(got[:, :H], ydt), y, ty + U[ydt] * (np.abs(y) + ty) + TINY[ydt], "y")
        assert (got[:, H:] == SENTINEL[ydt]).all()
    for b in {id(b): b for b in [xb, fb, ob, *wb.values()] + ([mb] if mb else []) + ([yb] if yb else [])}.values():
        b.free()


@pytest.mark.parametrize("H,xdt,fdt,ydt,mod_rows", [(2048, BF16, BF16, BF16, 1), (1000, F32, F16, F16, 397), (504, F16, F32, BF16, 5000)])
def test_gate_add_norm_large(tsn, rt, H, xdt, fdt, ydt, mod_rows):
    """traffic past the last-level cache (over 192 MiB), rows that several waves take in turn"""
    r = rng(H)
    size = lambda dt: 4 if dt == F32 else 2  # noqa: E731
    rows = (202 << 20) // (H * (2 * size(xdt) + size(fdt) + size(ydt))) + 1
    x, f = (enc(r.standard_normal((991, H)), dt)[np.arange(rows) % 991] for dt in (xdt, fdt))
    mod = (0.3 * r.standard_normal((-(-rows // mod_rows), 3 * H))).astype(np.float32)
    w = (1.0 + 0.1 * r.standard_normal(H)).astype(np.float32)
    c = dict(post=2, pre=1, x_scale=0.9, f_scale=1.1, mod_rows=mod_rows, gate=2, shift=0, scale=1, post_eps=1e-5, pre_eps=1e-6)
    xb, fb, mb, wb = rt.array(x), rt.array(f), rt.array(mod), rt.array(w)
    ob, yb = rt.array(np.full(x.shape, SENTINEL[xdt], NP[xdt])), rt.array(np.full(x.shape, SENTINEL[ydt], NP[ydt]))
    rt.gate_add_norm(tsn.gate_norm_spec(rows, H, xdt, fdt, ydt, chunks=3, **c), xb, fb, mb, ob, yb, post_w=wb, pre_w=wb)
    rt.sync()
    at = spread(rows, r)
    c.update(mod_rows=1, **{k: np.float64(np.float32(c[k])) for k in ("post_eps", "pre_eps")})
    ws = dict(post_w=w.astype(np.float64), pre_w=w.astype(np.float64))
    xo, ex, y, ty = gate_norm_ref(dec(x[at], xdt), dec(f[at], fdt), mod[at // mod_rows], c, ws)
    check(dec(ob.numpy()[at], xdt), xo, ex + U[xdt] * (np.abs(xo) + ex) + TINY[xdt], "x_out")
    check(dec(yb.numpy()[at], ydt), y, ty + U[ydt] * (np.abs(y) + ty) + TINY[ydt], "y")
    for b in (xb, fb, mb, wb, ob, yb):
        b.free()


def test_gate_add_norm_is_gate_add_then_adaln(tsn, rt):
    """without norm and weights on the block's side it is tsn_gate_add followed by tsn_adaln_ln"""
    r = rng(8)
    rows, H = 141, 1024
    x, f = (r.standard_normal((rows, H)).astype(np.float32) for _ in range(2))
    mod = (0.3 * r.standard_normal(3 * H)).astype(np.float32)
    xb, fb, mb, xo, y, x2, y2 = rt.array(x), rt.array(f), rt.array(mod), *(rt.empty((rows, H)) for _ in range(4))
    rt.gate_add_norm(tsn.gate_norm_spec(rows, H, post=0, pre=2, chunks=3, gate=2, shift=0, scale=1), xb, fb, mb, xo, y)
    rt.gate_add(xb, fb, mb, x2, rows, H, 0, 3, 2)
    rt.adaln_ln(x2, mb, y2, F32, rows, H, 0, 3, 0, 1e-5)
    rt.sync()
    assert rel_l2(xo.numpy(), x2.numpy()) <= 4 * E      # the same sum of two f32 products, fused or not
    # a norm of 1024 elements whose two sums are ordered differently: D of each side at most (see norm_ref)
    assert rel_l2(y.numpy(), y2.numpy()) <= 2 * E * (H / 64 + 24)


# ---------------------------------------------------------------- differential attention

def attn_ref(q, k, v, lam, w, ql, kl, causal, scale, lambda_init, eps, nh, nkv, hd, dt, heads=None):
    """(out, bound, live) in f64; q [B][Sq][nh*2*hd] and so on are the values that the elements stand for. heads: those
    that are computed, the others are not live"""
    B, Sq, _ = q.shape
    Sk = k.shape[1]
    out, tol, live = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape, bool)
    for b in range(B):
        n, m = int(np.clip(ql[b], 0, Sq)), int(np.clip(kl[b], 0, Sk))
        for h in range(nh) if heads is None else heads:
            live[b, :n, 2 * h * hd:2 * (h + 1) * hd] = True
        if n == 0 or m == 0:
            continue
        seen = np.arange(m)[None] <= (np.arange(n)[:, None] + (m - n) if causal else m)
        for h in range(nh) if heads is None else heads:
            g = h * nkv // nh
            L = lam[h if lam.shape[0] > 1 else 0]
            lm = np.exp(L[0] @ L[1]) - np.exp(L[2] @ L[3]) + lambda_init
            vv = v[b, :m, 2 * g * hd:2 * (g + 1) * hd]
            o, to = 0.0, 0.0
            for j, wt in ((0, 1.0), (1, lm)):
                qq, kk = (t[b, :c, (2 * i + j) * hd:(2 * i + j + 1) * hd] for t, c, i in ((q, n, h), (k, m, g)))
                s = np.where(seen, qq @ kk.T * scale, -np.inf)
                top = s.max(-1, keepdims=True)
                p = np.where(seen, np.exp(s - np.where(np.isfinite(top), top, 0.0)), 0.0)
                a = p / np.maximum(p.sum(-1, keepdims=True), 1e-300)
                # a score is a sum of hd products in f32, times scale*log2(e), less a reference as large as any
                # score: its error in the exponent; exp2 itself is good to 2^-22
                smax = np.abs(np.where(seen, s, 0.0)).max(-1, keepdims=True)
                es = E * (hd * (np.abs(qq) @ np.abs(kk).T * scale).max(-1, keepdims=True) + 6 * smax) + 2.0 ** -22
                # the probabilities are rounded once; numerator and denominator each carry these errors and the
                # f32 additions of m terms
                sign = 1.0 if j == 0 else -1.0
                o = o + sign * wt * (a @ vv)
                to = to + abs(wt) * (a @ np.abs(vv)) * (2 * (es + U[dt]) + 2 * E * (m + 16) + 64 * E)
            if w is not None:
                rms = np.sqrt((o * o).mean(-1, keepdims=True) + eps)
                er = (np.abs(o) * to + to * to).mean(-1, keepdims=True) / rms ** 2 + 16 * E   # relative, of 1/rms
                f = (1.0 - lambda_init) * w / rms
                o, to = o * f, np.abs(f) * (to + np.abs(o) * er)
            cols = np.s_[b, :n, 2 * h * hd:2 * (h + 1) * hd]
            out[cols], tol[cols] = o, to
    return out, tol + U[dt] * (np.abs(out) + tol) + TINY[dt], live


def attn_case(tsn, rt, dt, B, Sq, Sk, nh, nkv, hd, causal=False, ql=None, kl=None, lam_heads=1, norm=True, scale=None,
              lambda_init=0.5, pad=(0, 0, 0, 0), make=None, seed=0, junk=None, col=0, heads=None):
    """Runs one call and checks every element, the rows behind q_len and the columns around the heads. pad: elements
    behind the packed row of q, k, v, out; col: first column of each."""
    r = rng(seed + 31 * Sq + 7 * Sk + hd)
    wq, wk = 2 * nh * hd, 2 * nkv * hd
    q, k, v = r.standard_normal((B, Sq, wq)), r.standard_normal((B, Sk, wk)), r.standard_normal((B, Sk, wk))
    if make:
        q, k, v = make(r, q, k, v)
    q, k, v = (enc(t, dt) for t in (q, k, v))
    if junk is not None and kl is not None:   # what an earlier use of the buffer left behind the last key
        for b in range(B):
            k[b, kl[b]:], v[b, kl[b]:] = enc(junk, dt), enc(junk, dt)
    lam = (0.1 * r.standard_normal((lam_heads, 4, hd))).astype(np.float32)
    w = (1.0 + 0.1 * r.standard_normal(2 * hd)).astype(np.float32) if norm else None
    lds = [n + p for n, p in zip((wq, wk, wk, wq), pad)]
    bufs = [rt.array(strided(t.reshape(-1, t.shape[-1]), ld, dt, col)) for t, ld in zip((q, k, v), lds)]
    ob = rt.array(np.full((B * Sq, lds[3]), SENTINEL[dt], NP[dt]))
    lb, wb = rt.array(lam), rt.array(w) if norm else None
    qlb, klb = (None if t is None else rt.array(np.asarray(t, np.int32)) for t in (ql, kl))
    spec = tsn.diff_attn_spec(dt, B, Sq, Sk, nh, nkv, hd, causal=causal, scale=scale, lambda_init=lambda_init,
                              lam_heads=lam_heads, ldq=lds[0], ldk=lds[1], ldv=lds[2], ldo=lds[3])
    args = [At(t, col) for t in bufs] + [lb, wb, qlb, klb, At(ob, col)]
    rt.diff_attention(spec, *args)
    rt.sync()
    first = ob.numpy()
    ql2, kl2 = ([Sq] * B if ql is None else ql), ([Sk] * B if kl is None else kl)
    want, tol, live = attn_ref(*(dec(t, dt) for t in (q, k, v)), lam.astype(np.float64), None if w is None else w.astype(np.float64), ql2, kl2,
                               causal, np.float64(np.float32(hd ** -0.5 if scale is None else scale)), np.float64(np.float32(lambda_init)),
                               np.float64(np.float32(1e-5)), nh, nkv, hd, dt, heads)
    res = first[:, col:col + wq].reshape(B, Sq, wq)
    got = dec(res, dt)
    check(got[live], want[live], tol[live])
    behind = np.arange(Sq)[None, :] >= np.maximum(np.asarray(ql2), 0)[:, None]
    assert (res[behind] == SENTINEL[dt]).all(), "rows behind q_len were written"
    assert heads is not None or (live != behind[:, :, None]).all()
    assert (np.delete(first, np.s_[col:col + wq], 1) == SENTINEL[dt]).all(), "columns around the heads were written"
    rt.diff_attention(spec, *args)
    rt.sync()
    assert np.array_equal(first, ob.numpy()), "two runs differ"
    for t in bufs + [ob, lb] + [t for t in (wb, qlb, klb) if t is not None]:
        t.free()
    return got[live], want[live]


SHAPES = [
    # B Sq Sk nh nkv causal
    (1, 1, 1, 1, 1, False), (1, 1, 2, 2, 1, True), (2, 1, 33, 4, 4, False), (1, 3, 31, 2, 2, True), (1, 5, 4, 3, 1, True),
    (2, 17, 64, 2, 2, False), (1, 64, 65, 4, 2, True), (2, 63, 200, 6, 2, True), (1, 130, 129, 2, 1, False),
    (1, 257, 257, 3, 3, True), (1, 1, 4097, 4, 2, False), (3, 1, 1000, 8, 2, True), (1, 4, 2500, 4, 1, True),
    (1, 33, 1030, 2, 2, False), (2, 397, 397, 4, 4, False), (1, 700, 900, 2, 2, True), (5, 2, 95, 3, 3, True), (1, 16, 8200, 2, 1, True),
]


@pytest.mark.parametrize("hd", [64, 32])
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("B,Sq,Sk,nh,nkv,causal", SHAPES)
def test_diff_attention(tsn, rt, dt, hd, B, Sq, Sk, nh, nkv, causal):
    got, want = attn_case(tsn, rt, dt, B, Sq, Sk, nh, nkv, hd, causal, lam_heads=nh if Sq % 2 else 1, norm=Sk % 3 != 0)
    if Sk >= 1000 and not causal:
        # the rounding of the result and those of the probabilities are independent: u/sqrt(3) each at most (the
        # two maps' add as the squares of their shares of the difference); 2u is over twice their joint size
        assert rel_l2(got, want) <= 2 * U[dt]


# sizes at which the work is cut in each way, and the cuts fall inside tiles
CUTS = [
    # B Sq Sk nh nkv causal kl heads
    (70, 1, 6000, 2, 1, True, "ragged", None),         # one row of more than 64 samples: shared out by the lengths
    (66, 2, 6000, 2, 1, False, "some empty", None),
    (130, 1, 4000, 2, 1, True, "ragged", None),        # a workgroup each
    (70, 3, 1500, 2, 1, False, "some empty", None),
    (1, 1, 70000, 2, 1, False, None, None),            # one row over a long cache
    (2, 40, 6000, 4, 1, True, "ragged", None),         # several tiles of few rows
    (1, 1000, 8192, 4, 4, True, None, (0, 3)),         # wide tiles shared out
    (2, 600, 9000, 2, 2, False, "ragged", None),
    (1, 1300, 3000, 50, 50, False, None, (0, 24, 46, 49)),   # the tiles behind the last full round shared out
    (3, 1000, 2500, 24, 24, False, "ragged", (0, 11, 23)),
    (1, 2500, 2500, 8, 8, True, None, (2, 7)),         # causal tiles, heads round the XCDs
    (4, 500, 500, 6, 2, True, "ragged", (0, 5)),
    (5, 1300, 1500, 40, 10, True, "ragged", (0, 23, 39)),      # causal tiles by length: all resident at once
    (33, 700, 700, 16, 8, True, "some empty", (0, 9, 15)),     # more of them, samples without rows and without keys
    (3, 1500, 400, 48, 48, True, "ragged", (0, 47)),           # more rows than keys: tiles without keys
    (2, 4100, 4100, 12, 2, True, None, (0, 11)),               # heads that do not go round the XCDs
    (70, 330, 330, 16, 8, True, "some empty", (0, 15)),        # more samples than are ranked
]


@pytest.mark.parametrize("dt,hd", [(F16, 64), (BF16, 32)])
@pytest.mark.parametrize("B,Sq,Sk,nh,nkv,causal,kl,heads", CUTS)
def test_diff_attention_cuts(tsn, rt, dt, hd, B, Sq, Sk, nh, nkv, causal, kl, heads):
    r = rng(B + Sq)
    lens = None if kl is None else [int(t) for t in r.integers(Sk // 4, Sk + 1, B)]
    ql = None
    if kl == "some empty":
        lens[3], lens[B - 5], lens[B - 1] = 0, 1, 0
        ql = [int(t) for t in r.integers(0, Sq + 1, B)]
    attn_case(tsn, rt, dt, B, Sq, Sk, nh, nkv, hd, causal, ql, lens, junk=None if kl is None else np.nan, heads=heads)


@pytest.mark.parametrize("hd", [64, 32])
@pytest.mark.parametrize("dt,junk", [(F16, np.nan), (BF16, np.inf)])
@pytest.mark.parametrize("B,Sq,Sk,nh,nkv,causal,ql,kl", [
    (3, 40, 300, 2, 2, False, [40, 0, 7], [300, 300, 0]),             # no rows; no keys
    (4, 70, 70, 4, 2, True, [70, 33, 1, 64], [70, 33, 1, 64]),        # prompts of unequal length
    (3, 50, 90, 2, 1, True, [50, 50, 20], [10, 63, 90]),              # rows before the first key: empty
    (4, 1, 1500, 4, 2, True, [1, 1, 1, 1], [1500, 1, 0, 767]),
    (2, 1, 513, 8, 8, False, None, [512, 513]),
    (3, 140, 210, 4, 2, True, [0, 139, 140], None),
    (3, 130, 260, 2, 2, False, [129, 130, 64], [65, 64, 1]),
    (2, 5, 3000, 2, 1, True, [5, 3], [2, 2999]),
    (2, 33, 128, 1, 1, False, [-5, 99], [200, -1]),                   # out of range: taken as none and all
])
def test_diff_attention_lengths(tsn, rt, dt, junk, hd, B, Sq, Sk, nh, nkv, causal, ql, kl):
    attn_case(tsn, rt, dt, B, Sq, Sk, nh, nkv, hd, causal, ql, [min(max(t, 0), Sk) for t in kl] if kl and (min(kl) < 0 or max(kl) > Sk) else kl,
              junk=junk)
    if kl and (min(kl) < 0 or max(kl) > Sk):   # the same with the lengths as they are
        attn_case(tsn, rt, dt, B, Sq, Sk, nh, nkv, hd, causal, ql, kl)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("Sq,pad,col", [(1, (8, 16, 24, 32), 8), (90, (8, 16, 24, 32), 8), (90, (0, 256, 256, 0), 0),
                                        (1, (1, 3, 5, 7), 1), (90, (1, 3, 5, 7), 1), (34, (4, 4, 4, 4), 4), (34, (0, 0, 0, 1), 0)])
def test_diff_attention_strides(tsn, rt, dt, Sq, pad, col):
    attn_case(tsn, rt, dt, 2, Sq, 200, 4, 2, 64, True, kl=[200, 150], junk=np.nan, pad=pad, col=col)


@pytest.mark.parametrize("hd", [64, 32])
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("kind", ["rising", "falling", "spike", "equal", "zero_scale", "large"])
@pytest.mark.parametrize("Sq", [2, 96])
def test_diff_attention_scores(tsn, rt, dt, hd, kind, Sq):
    """the running maximum moves with every key block, never, once at the end, and by hundreds"""
    def make(r, q, k, v):
        S = k.shape[1]
        ramp = np.linspace(0.0, 6.0, S)[None, :, None]
        if kind in ("rising", "falling"):
            q, k = np.abs(q), np.abs(k) * (ramp if kind == "rising" else ramp[:, ::-1])
        elif kind == "spike":
            k[:, S - 2] = 4.0 * np.sign(q[:, :1, :k.shape[2]])[:, 0]
        elif kind == "equal":
            k[:] = k[:, :1]
        elif kind == "large":
            q, k = 12.0 * q, 12.0 * k
        return q, k, v

    attn_case(tsn, rt, dt, 1, Sq, 700, 2, 2, hd, make=make, scale=0.0 if kind == "zero_scale" else None)


@pytest.mark.parametrize("lambda_init", [0.0, 0.2, 0.8])
def test_diff_attention_lambda(tsn, rt, lambda_init):
    attn_case(tsn, rt, F16, 2, 40, 300, 4, 4, 64, lam_heads=4, lambda_init=lambda_init)


@pytest.mark.parametrize("hd", [64, 32])
@pytest.mark.parametrize("B,Sq,Sk,nkv,pad", [(2, 5, 300, 2, 0), (2, 5, 300, 2, 1), (2, 3, 9000, 1, 0), (8, 1300, 700, 16, 0), (2, 900, 3000, 2, 0)])
def test_diff_attention_no_keys_no_eps(tsn, rt, hd, B, Sq, Sk, nkv, pad):
    """rows that see no key are zeros with an eps of 0 too: a sample without keys, and causal rows before the first"""
    w = 2 * nkv * hd
    r = rng(Sk + hd)
    q = rt.array(enc(r.standard_normal((B * Sq, w + pad)), F16))
    k = rt.array(enc(r.standard_normal((B * Sk, w)), F16))
    lam, nw = rt.array(np.zeros((1, 4, hd), np.float32)), rt.array(np.ones(2 * hd, np.float32))
    kl = [0] + [Sk] * (B - 2) + [Sq - 2]
    klb, o = rt.array(np.asarray(kl, np.int32)), rt.array(np.full((B * Sq, w), np.nan, np.float16))
    rt.diff_attention(tsn.diff_attn_spec(F16, B, Sq, Sk, nkv, nkv, hd, causal=True, eps=0.0, ldq=w + pad), q, k, k, lam, nw, None, klb, o)
    rt.sync()
    got = o.numpy().reshape(B, Sq, w)
    for b in range(B):
        empty = max(0, Sq - min(kl[b], Sk))   # lengths past Sk are Sk
        assert (got[b, :empty] == 0).all()
        assert np.isfinite(got[b, empty:]).all() and (got[b, empty + 1:] != 0).any(-1).all()
    for t in (q, k, lam, nw, klb, o):
        t.free()


def test_diff_attention_far_offsets(tsn, rt):
    """samples and rows of a cache that lie more than 2^32 bytes from its start"""
    dt, hd, Sk, nh = F16, 64, 130, 2
    wk, far = 2 * nh * hd, (1 << 31) + 4096           # elements between the two samples
    r = rng(77)
    big = rt.empty((far + Sk * 2 * wk,), np.float16)
    rows = r.standard_normal((2, Sk, 2 * wk)).astype(np.float16)   # k | v
    for b in range(2):
        part = np.ascontiguousarray(rows[b])
        tsn.call("tsn_upload", rt.h, big.offset(b * far), tsn.ptr(part), part.nbytes)
    q = r.standard_normal((2, 3, wk)).astype(np.float16)
    lam = (0.1 * r.standard_normal((1, 4, hd))).astype(np.float32)
    qb, lb, ob = rt.array(q), rt.array(lam), rt.empty((2, 3, wk), np.float16)
    spec = tsn.diff_attn_spec(dt, 2, 3, Sk, nh, nh, hd, causal=True, lambda_init=0.5, ldk=2 * wk, ldv=2 * wk, bsk=far, bsv=far)
    rt.diff_attention(spec, qb, big, At(big, wk), lb, None, None, None, ob)
    rt.sync()
    want, tol, _ = attn_ref(q.astype(np.float64), rows[..., :wk].astype(np.float64), rows[..., wk:].astype(np.float64), lam.astype(np.float64),
                            None, [3, 3], [Sk, Sk], True, hd ** -0.5, 0.5, 1e-5, nh, nh, hd, dt)
    check(ob.numpy().astype(np.float64), want, tol)
    for t in (big, qb, lb, ob):
        t.free()


def test_diff_attention_far_rows(tsn, rt):
    """one sample whose rows reach past 2^32 bytes"""
    dt, hd, Sk, ld = BF16, 32, 600, 1 << 22
    r = rng(78)
    big = rt.empty((Sk * ld - ld + 256,), np.uint16)
    rows = enc(r.standard_normal((Sk, 128)), dt)      # k | v of one head
    for j in range(Sk):
        part = np.ascontiguousarray(rows[j])
        tsn.call("tsn_upload", rt.h, big.offset(j * ld), tsn.ptr(part), part.nbytes)
    lam = (0.1 * r.standard_normal((1, 4, hd))).astype(np.float32)
    for Sq in (1, 70):
        q = enc(r.standard_normal((1, Sq, 64)), dt)
        qb, lb, ob = rt.array(q), rt.array(lam), rt.empty((1, Sq, 64), np.uint16)
        spec = tsn.diff_attn_spec(dt, 1, Sq, Sk, 1, 1, hd, lambda_init=0.5, ldk=ld, ldv=ld)
        rt.diff_attention(spec, qb, big, At(big, 64), lb, None, None, None, ob)
        rt.sync()
        want, tol, _ = attn_ref(dec(q, dt), dec(rows[None, :, :64], dt), dec(rows[None, :, 64:], dt), lam.astype(np.float64), None,
                                [Sq], [Sk], False, np.float64(np.float32(hd ** -0.5)), 0.5, 1e-5, 1, 1, hd, dt)
        check(dec(ob.numpy(), dt), want, tol)
    big.free()


def test_block_operators_allocations(tsn):
    """rope_axes and gate_add_norm take no device memory, diff_attention the runtime's scratch once: a second call of the
    same or a smaller size allocates nothing"""
    r = rng(9)
    with tsn.Runtime(0) as rt2:
        q, k = rt2.array(enc(r.standard_normal((1, 4, 256)), F16)), rt2.array(enc(r.standard_normal((1, 9000, 256)), F16))
        lam, o = rt2.array(np.zeros((1, 4, 64), np.float32)), rt2.empty((1, 4, 256), np.float16)
        pos, y = rt2.array(np.zeros((4, 1), np.int32)), rt2.empty((4, 256), np.float16)
        before = rt2.alloc_stats()
        rt2.rope_axes(tsn.rope_axes_spec(F16, 4, 4, 64, (64,), (1e4,)), q, pos, y)
        rt2.gate_add_norm(tsn.gate_norm_spec(4, 256, F16, F16, F16), q, y, None, q, y)
        assert rt2.alloc_stats() == before
        rt2.diff_attention(tsn.diff_attn_spec(F16, 1, 4, 9000, 2, 2, 64), q, k, k, lam, None, None, None, o)
        once = rt2.alloc_stats()
        assert once[0] <= before[0] + 1
        for Sk in (9000, 5000):
            rt2.diff_attention(tsn.diff_attn_spec(F16, 1, 4, Sk, 2, 2, 64), q, k, k, lam, None, None, None, o)
        rt2.sync()
        assert rt2.alloc_stats() == once


def test_two_runtimes_at_once(tsn, rt):
    """two streams with calls in flight together: each has its own workspace, both give what they give alone"""
    r = rng(10)
    with tsn.Runtime(0) as rt2:
        sides = []
        for R, Sk in ((rt, 9001), (rt2, 7003)):
            q, k, v = (R.array(enc(r.standard_normal((1, n, 256)), F16)) for n in (4, Sk, Sk))
            lam, o = R.array(np.zeros((1, 4, 64), np.float32)), R.empty((1, 4, 256), np.float16)
            sides.append((R, tsn.diff_attn_spec(F16, 1, 4, Sk, 2, 2, 64, lambda_init=0.5), (q, k, v, lam, None, None, None, o)))
        alone = []
        for R, s, a in sides:
            R.diff_attention(s, *a)
            R.sync()
            alone.append(a[-1].numpy())
        for _ in range(20):
            for R, s, a in sides:
                R.diff_attention(s, *a)
        for (R, _, a), w in zip(sides, alone):
            R.sync()
            assert np.array_equal(a[-1].numpy(), w)
        for t in sides[0][2]:
            if t is not None:
                t.free()


# ---------------------------------------------------------------- together

def test_attention_half_block(tsn, rt):
    """A block's attention half as a program runs it: q|k heads of f16 q|k|v rows turned in place by (time, y, x), the
    difference of the maps, the out-projection, and the block's end. Against the same graph in 64 bits on the same
    rounded inputs: every f16 rounding on the way (turned q|k, probabilities, attention rows, the branch's operands)
    is at most 2^-11 relative and they add up as squares; eight of them are 2^-11 * sqrt(8) < 1.4e-3 of the branch."""
    B, S, H, nh, hd = 2, 397, 1024, 8, 64
    r = rng(11)
    qkv = enc(r.standard_normal((B * S, 3 * H)), F16)
    pos = np.stack([np.arange(S) // 64, (np.arange(S) // 8) % 8, np.arange(S) % 8], 1).astype(np.int32)
    lam = (0.1 * r.standard_normal((1, 4, hd))).astype(np.float32)
    w = (1.0 + 0.1 * r.standard_normal(2 * hd)).astype(np.float32)
    W = (r.standard_normal((H, H)) / 32.0).astype(np.float16)
    x = r.standard_normal((B * S, H)).astype(np.float32)
    mod = (0.3 * r.standard_normal((B, 3 * H))).astype(np.float32)
    pw, qw = ((1.0 + 0.1 * r.standard_normal(H)).astype(np.float32) for _ in range(2))
    kl = [S, S - 60]
    d = {n: rt.array(t) for n, t in dict(qkv=qkv, pos=pos, lam=lam, w=w, W=W, x=x, mod=mod, pw=pw, qw=qw, kl=np.array(kl, np.int32)).items()}
    o, f, y = rt.empty((B * S, H), np.float16), rt.empty((B * S, H)), rt.empty((B * S, H), np.float16)
    dims, bases = (16, 24, 24), (1e4, 1e2, 1e2)
    rt.rope_axes(tsn.rope_axes_spec(F16, B * S, 4 * nh, hd, dims, bases, ldx=3 * H, ldy=3 * H, pos_rows=S), d["qkv"], d["pos"], d["qkv"])
    rt.diff_attention(tsn.diff_attn_spec(F16, B, S, S, nh, nh, hd, lambda_init=0.5, ldq=3 * H, ldk=3 * H, ldv=3 * H),
                      d["qkv"], At(d["qkv"], H), At(d["qkv"], 2 * H), d["lam"], d["w"], None, d["kl"], o)
    rt.gemm(F16, d["W"], o, F16, f, F32, None, B * S, H, H)
    rt.gate_add_norm(tsn.gate_norm_spec(B * S, H, F32, F32, F16, post=1, pre=2, chunks=3, mod_rows=S, gate=2, shift=0, scale=1),
                     d["x"], f, d["mod"], d["x"], y, post_w=d["pw"], pre_w=d["qw"])
    rt.sync()
    full = dec(qkv, F16).reshape(B * S, 3, 2 * nh, hd)
    p2 = np.tile(pos, (B, 1))
    qk = [rope_ref(full[:, j], p2, dims, bases, (1.0,) * 3, False, False).reshape(B, S, H) for j in (0, 1)]
    ref, _, _ = attn_ref(qk[0], qk[1], full[:, 2].reshape(B, S, H), lam.astype(np.float64), w.astype(np.float64), [S] * B, kl, False,
                         hd ** -0.5, 0.5, np.float64(np.float32(1e-5)), nh, nh, hd, F16)
    fr = ref.reshape(B * S, H) @ W.astype(np.float64).T
    c = dict(post=1, pre=2, x_scale=1.0, f_scale=1.0, mod_rows=S, gate=2, shift=0, scale=1, post_eps=1e-5, pre_eps=1e-5)
    xo, _, yr, _ = gate_norm_ref(x.astype(np.float64), fr, mod.astype(np.float64), c, dict(post_w=pw.astype(np.float64), pre_w=qw.astype(np.float64)))
    assert rel_l2(f.numpy(), fr) <= 1.4e-3
    assert rel_l2(d["x"].numpy() - x, xo - x) <= 1.4e-3
    assert rel_l2(y.numpy().astype(np.float64), yr) <= 1.4e-3
    for t in [*d.values(), o, f, y]:
        t.free()
