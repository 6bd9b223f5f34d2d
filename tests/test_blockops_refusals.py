"""Refusals of the block operators (tsn_rope_axes, tsn_diff_attention, tsn_gate_add_norm), without a GPU: the entry
points check their arguments before the runtime handle, so a call that passes every check ends at the null
handle and any other names what is wrong. Nothing is launched and no pointer is followed."""
import ctypes

import numpy as np
import pytest

NULL_RT = "null runtime handle"
BASE = 1 << 40   # an address that nothing follows


def _call(tsn, name, *args):
    rc = getattr(tsn.lib(), name)(None, *args)
    return rc, tsn.lib().tsn_last_error().decode()


def _set(spec, kw):
    for k, v in kw.items():
        if isinstance(v, tuple):
            getattr(spec, k)[v[0]] = v[1]
        else:
            setattr(spec, k, v)
    return spec


def rope(tsn, x=BASE, pos=BASE + (1 << 36), y=BASE + (1 << 35), **kw):
    s = tsn.rope_axes_spec(tsn.F16, 10, 4, 64, (16, 24, 24), (1e4, 100.0, 100.0))
    return _call(tsn, "tsn_rope_axes", _set(s, kw), x, pos, y)


@pytest.mark.parametrize("kw,word", [
    (dict(), NULL_RT),
    (dict(y=BASE), NULL_RT),                                   # in place
    (dict(x=None), "null tensor"), (dict(pos=None), "null tensor"), (dict(y=None), "null tensor"),
    (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"),
    (dict(rows=0), "empty"), (dict(nh=0), "empty"), (dict(hd=0), "empty"),
    (dict(hd=63), "even"), (dict(hd=258), "256"),
    (dict(n_axes=0), "axes"), (dict(n_axes=5), "axes"),
    (dict(rows=1 << 31), "rows"), (dict(rows=(1 << 31) - 1, dtype=0, ldx=(1 << 31) + 8, x=1 << 20, y=BASE), "overlap"),
    (dict(dim=(1, 23)), "even"), (dict(dim=(1, 26)), "more than hd"), (dict(dim=(0, 0xFFFFFFFE)), "more than hd"),
    (dict(base=(0, 0.0)), "base"), (dict(base=(2, -1.0)), "base"), (dict(base=(1, float("nan"))), "base"),
    (dict(fscale=(0, float("inf"))), "finite"),
    (dict(ldx=255), "stride"), (dict(ldy=100), "stride"),
    (dict(y=BASE + 2), "overlap"), (dict(y=BASE, ldy=300), "overlap"), (dict(y=BASE + 9 * 512), "overlap"),
    (dict(y=BASE + 10 * 512), NULL_RT),                        # right behind
    (dict(ldx=512, ldy=512, y=BASE + 512), NULL_RT),           # other columns of the same rows
    (dict(ldx=512, ldy=512, x=BASE + 512, y=BASE), NULL_RT),
    (dict(ldx=512, ldy=512, y=BASE + 510), "overlap"),
    (dict(x=BASE + 1), "aligned"), (dict(pos=BASE + (1 << 36) + 2), "aligned"),
    (dict(pos=BASE + (1 << 35) + 64), "overlaps pos"),
])
def test_rope_axes(tsn, kw, word):
    rc, msg = rope(tsn, **kw)
    assert rc == 1 and word in msg, (rc, msg)


def attn(tsn, q=BASE, k=BASE + (1 << 36), v=BASE + (2 << 36), lam=BASE + (3 << 36), w=BASE + (4 << 36), ql=None, kl=None,
         out=BASE + (5 << 36), **kw):
    s = tsn.diff_attn_spec(tsn.F16, 2, 40, 50, 8, 4, 64)
    return _call(tsn, "tsn_diff_attention", _set(s, kw), q, k, v, lam, w, ql, kl, out)


@pytest.mark.parametrize("kw,word,code", [
    (dict(), NULL_RT, 1), (dict(w=None, eps=float("nan")), NULL_RT, 1), (dict(lam_heads=8), NULL_RT, 1),
    (dict(q=None), "null tensor", 1), (dict(k=None), "null tensor", 1), (dict(v=None), "null tensor", 1),
    (dict(lam=None), "null tensor", 1), (dict(out=None), "null tensor", 1),
    (dict(dtype=0), "dtype", 1), (dict(dtype=7), "dtype", 1),
    (dict(B=0), "empty", 1), (dict(Sq=0), "empty", 1), (dict(Sk=0), "empty", 1), (dict(nh=0), "empty", 1), (dict(nkv=0), "empty", 1),
    (dict(hd=48), "32 or 64", 3), (dict(hd=128), "32 or 64", 3),
    (dict(nkv=3), "multiple", 1), (dict(nkv=16), "multiple", 1),
    (dict(lam_heads=0), "lambda vectors", 1), (dict(lam_heads=4), "lambda vectors", 1),
    (dict(scale=float("nan")), "scale", 1), (dict(scale=-0.1), "scale", 1),
    (dict(lambda_init=1.0), "lambda_init", 1), (dict(lambda_init=-0.1), "lambda_init", 1), (dict(lambda_init=float("nan")), "lambda_init", 1),
    (dict(eps=-1.0), "eps", 1),
    (dict(nh=8192, nkv=8192), "launch grid", 1), (dict(B=1 << 20, Sq=1 << 20), "launch grid", 1), (dict(Sk=1 << 30), "launch grid", 1),
    (dict(ldq=1023), "row stride", 1), (dict(ldk=511), "row stride", 1), (dict(ldv=500), "row stride", 1), (dict(ldo=1000), "row stride", 1),
    (dict(ldk=(1 << 22) + 8), "row stride", 1), (dict(bsk=1 << 40), "sample stride", 1),
    (dict(bso=39 * 1024), "samples of out", 1), (dict(bso=1024, ldo=2048), NULL_RT, 1),
    (dict(B=1 << 23, Sq=1, nh=1, nkv=1, bsq=(1 << 40) - 8, bsk=1 << 8), "overlaps an input", 1),
    (dict(q=BASE + 1), "aligned", 1), (dict(lam=BASE + (3 << 36) + 2), "aligned", 1),
    (dict(out=BASE), "overlaps an input", 1), (dict(out=BASE + (1 << 36) + 1024), "overlaps an input", 1),
    (dict(out=BASE + (2 << 36) - 2048), "overlaps an input", 1),
    (dict(out=BASE + 2048, ldo=2048, ldq=2048), NULL_RT, 1),                        # other columns of q's rows
    (dict(out=BASE + 2046, ldo=2048, ldq=2048), "overlaps an input", 1),
    (dict(out=BASE + (4 << 36)), "overlaps lam", 1), (dict(kl=BASE + (5 << 36)), "overlaps lam", 1),
])
def test_diff_attention(tsn, kw, word, code):
    rc, msg = attn(tsn, **kw)
    assert rc == code and word in msg, (rc, msg)


def norm(tsn, x=BASE, f=BASE + (1 << 36), mod=BASE + (2 << 36), pw=None, pb=None, qw=None, qb=None, xo=BASE + (3 << 36),
         y=BASE + (4 << 36), **kw):
    s = tsn.gate_norm_spec(20, 100, chunks=3, gate=2, shift=0, scale=1, mod_rows=5)
    return _call(tsn, "tsn_gate_add_norm", _set(s, kw), x, f, mod, pw, pb, qw, qb, xo, y)


@pytest.mark.parametrize("kw,word,code", [
    (dict(), NULL_RT, 1), (dict(y=None), NULL_RT, 1), (dict(mod=None, gate=-1, shift=-1, scale=-1), NULL_RT, 1),
    (dict(xo=BASE), NULL_RT, 1), (dict(y=BASE + (1 << 36)), NULL_RT, 1),            # in place of x, of f
    (dict(x=None), "null tensor", 1), (dict(f=None), "null tensor", 1), (dict(xo=None), "null tensor", 1),
    (dict(x_dtype=3), "dtype", 1), (dict(f_dtype=-1), "dtype", 1), (dict(y_dtype=9), "dtype", 1),
    (dict(post=3), "norm kind", 1), (dict(pre=-1), "norm kind", 1),
    (dict(rows=0), "empty", 1), (dict(H=0), "empty", 1), (dict(H=16385), "16384", 3),
    (dict(x_scale=float("nan")), "scales", 1), (dict(f_scale=float("inf")), "scales", 1),
    (dict(rows=1 << 31), "rows", 1), (dict(rows=(1 << 31) - 1, ldf=(1 << 31) + 8, f=1 << 20, xo=BASE, y=None, mod=None, gate=-1, shift=-1, scale=-1), "x_out overlaps f", 1),
    (dict(post_eps=-1.0), "eps", 1), (dict(pre_eps=float("nan")), "eps", 1),
    (dict(gate=3), "chunk", 1), (dict(shift=-2), "chunk", 1), (dict(scale=7), "chunk", 1), (dict(mod=None), "chunk", 1),
    (dict(ldx=99), "stride", 1), (dict(ldf=1), "stride", 1), (dict(ldo=99), "stride", 1), (dict(ldy=50), "stride", 1),
    (dict(x=BASE + 2), "aligned", 1), (dict(pw=BASE + (5 << 36) + 1), "aligned", 1),
    (dict(xo=BASE + 4), "x_out must be x", 1), (dict(xo=BASE, ldo=120), "x_out must be x", 1), (dict(xo=BASE + (1 << 36)), "overlaps f", 1),
    (dict(y=BASE + (1 << 36), y_dtype=1), "y must be f", 1), (dict(y=BASE), "overlaps x", 1), (dict(y=BASE + (3 << 36)), "overlaps x", 1),
    (dict(y=BASE + (2 << 36)), "overlaps mod", 1), (dict(pw=BASE + (3 << 36)), "overlaps mod", 1),
])
def test_gate_add_norm(tsn, kw, word, code):
    rc, msg = norm(tsn, **kw)
    assert rc == code and word in msg, (rc, msg)


def test_null_specs(tsn):
    assert _call(tsn, "tsn_rope_axes", None, None, None, None) == (1, "rope_axes: null spec")
    assert _call(tsn, "tsn_diff_attention", None, *[None] * 8) == (1, "diff_attention: null spec")
    assert _call(tsn, "tsn_gate_add_norm", None, *[None] * 9) == (1, "gate_add_norm: null spec")


class Fake:
    def __init__(self, n, itemsize):
        self.nbytes, self.p = n * itemsize, ctypes.c_void_p(BASE)


def test_wrappers_check_array_sizes(tsn):
    """device arrays shorter than the spec reaches are refused before the library is called"""
    rt = tsn.Runtime.__new__(tsn.Runtime)
    rt.h = None
    s = tsn.rope_axes_spec(tsn.F16, 10, 4, 64, (16, 24), (1e4, 100.0), ldx=300, pos_rows=5)
    ok = dict(x=Fake(9 * 300 + 256, 2), pos=Fake(10, 4), y=Fake(2560, 2))
    for k in ok:
        bad = dict(ok, **{k: Fake(ok[k].nbytes // 2 - 1, 2)})
        with pytest.raises(ValueError):
            rt.rope_axes(s, bad["x"], bad["pos"], bad["y"])
    with pytest.raises(ValueError):
        rt.rope_axes(s, ok["x"], None, ok["y"])
    with pytest.raises(TypeError):
        rt.rope_axes(s, np.zeros(9999), ok["pos"], ok["y"])
    s = tsn.diff_attn_spec(tsn.BF16, 2, 3, 7, 4, 2, 32, bsk=1000, lam_heads=4)
    ok = dict(q=Fake(2 * 3 * 256, 2), k=Fake(1000 + 7 * 128, 2), v=Fake(2 * 7 * 128, 2), lam=Fake(4 * 4 * 32, 4),
              norm_w=Fake(64, 4), q_len=Fake(2, 4), kv_len=Fake(2, 4), out=Fake(2 * 3 * 256, 2))
    for k in ok:
        bad = dict(ok, **{k: Fake(ok[k].nbytes // 2 - 1, 2)})
        with pytest.raises(ValueError):
            rt.diff_attention(s, **bad)
    s = tsn.gate_norm_spec(11, 96, y_dtype=tsn.F16, chunks=2, gate=1, mod_rows=4, ldx=100)
    ok = dict(x=Fake(10 * 100 + 96, 4), f=Fake(11 * 96, 4), mod=Fake(3 * 2 * 96, 4), x_out=Fake(11 * 96, 4),
              y=Fake(11 * 96, 2), post_w=Fake(96, 4), post_b=Fake(96, 4), pre_w=Fake(96, 4), pre_b=Fake(96, 4))
    for k in ok:
        bad = dict(ok, **{k: Fake(ok[k].nbytes // 2 - 1, 2)})
        with pytest.raises(ValueError):
            rt.gate_add_norm(s, **bad)
    gone = Fake(96, 4)   # a freed array is not an absent one
    gone.p = None
    with pytest.raises(ValueError, match="freed"):
        rt.gate_add_norm(s, **dict(ok, post_w=gone))
    with pytest.raises(ValueError):
        tsn.rope_axes_spec(tsn.F32, 1, 1, 64, (8,) * 5, (1e4,) * 5)
    with pytest.raises(ValueError):
        tsn.rope_axes_spec(tsn.F32, 1, 1, 64, (8, 8), (1e4,))


@pytest.mark.parametrize("kw,word", [
    # one sample: its stride is not taken
    (dict(B=1, bsq=5, out=BASE + 2048, ldo=2048, ldq=2048), NULL_RT),
    (dict(B=1, bso=77, out=BASE + 2048, ldo=2048, ldq=2048), NULL_RT),
    (dict(B=1, bsq=5, out=BASE + 2046, ldo=2048, ldq=2048), "overlaps an input"),
    # one row: its stride is not taken (q and out of every sample in one row of 2048)
    (dict(Sq=1, ldq=1032, ldo=1024, bsq=2048, bso=2048, out=BASE + 2048), NULL_RT),
    (dict(Sq=1, ldq=1032, ldo=1024, bsq=2048, bso=2048, out=BASE + 2000), "overlaps an input"),
    # samples between each other's rows: [row][sample][q | out]
    (dict(ldq=4096, ldo=4096, bsq=2048, bso=2048, out=BASE + 2048), NULL_RT),
    (dict(ldq=4096, ldo=4096, bsq=2048, bso=2048, out=BASE + 2040), "overlaps an input"),
    (dict(ldq=4096, ldo=4096, bsq=2048, bso=2048, out=BASE + 2056), "overlaps an input"),
    (dict(ldq=4096, ldo=4096, bsq=2048, bso=2040, out=BASE + 2048), "overlaps an input"),
    (dict(ldq=2048, ldo=4096, out=BASE + 2048), NULL_RT),             # every other row of q's
    (dict(ldq=2048, ldo=4096, bso=40 * 4096 + 1024, out=BASE + 2048), "overlaps an input"),
])
def test_diff_attention_shared_rows(tsn, kw, word):
    """out in the same buffer as q is taken wherever no element is shared, whatever strides are not used"""
    rc, msg = attn(tsn, **kw)
    assert rc == 1 and word in msg, (rc, msg)


def test_windows_brute_force(tsn):
    """q and out a few rows and samples in one small buffer, against the elements themselves: no call is taken in which two
    of out's elements, or one of out's and one of q's, are the same"""
    r = np.random.default_rng(3)
    taken = 0
    for _ in range(4000):
        B, Sq, nh = int(r.integers(1, 4)), int(r.integers(1, 4)), 1
        w = 64   # 2 * nh * hd of width 32
        ldq, ldo = (int(w * r.integers(1, 5) + r.choice([0, 0, 0, 8])) for _ in range(2))
        bsq, bso = (int(w * r.integers(1, 12)) for _ in range(2))
        at = int(w * r.integers(0, 6) + r.choice([0, 0, 0, 4, 60]))
        q = {b * bsq + i * ldq + c for b in range(B) for i in range(Sq) for c in range(w)}
        o = [at + b * bso + i * ldo + c for b in range(B) for i in range(Sq) for c in range(w)]
        rc, msg = attn(tsn, B=B, Sq=Sq, nh=nh, nkv=1, hd=32, ldq=ldq, ldo=ldo, bsq=bsq, bso=bso, out=BASE + 2 * at)
        if NULL_RT in msg:
            taken += 1
            assert len(set(o)) == len(o) and not q & set(o), (B, Sq, ldq, ldo, bsq, bso, at)
        else:
            assert "overlap" in msg, msg
    assert taken > 400
