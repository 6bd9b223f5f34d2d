"""tsn_diff_attention where its work is cut: no key may be lost or counted twice. Evenly spread values average out over
long caches, so here every 32 (128) keys have a column of V to themselves (the blocks take the columns in turn): a result's element
is the weight of a few blocks, and one of them less or more is further off than the tolerance. That this is so is shown on
the CPU, by leaving blocks out of the reference and repeating them."""
import numpy as np
import pytest

from conftest import rng
from test_gpu_blockops import BF16, CUTS, F16, NP, SENTINEL, attn_ref, check, dec, enc


def block_of(Sk):
    """keys of a block: those of a wave in a unit of 128, and over the longest cache, as the bound grows with its length, all
    of a unit (the work is cut between units)"""
    return 32 if Sk < 20000 else 128


LAMBDA = -0.9   # both maps add up: a block that one of them loses is not made good by the other
MORE = [
    # B Sq Sk nh nkv causal kl heads: lengths in long caches, and a size for each kernel that is in one piece
    (2, 5, 3000, 2, 1, True, [2, 2999], None),
    (3, 1, 4097, 4, 2, True, [4097, 4096, 65], None),
    (8, 40, 3000, 16, 16, False, "ragged", (0, 15)),
    (1, 1300, 2049, 64, 64, True, None, (0, 63)),
]


def cut_case(case, hd, dt):
    """inputs of a case, as device elements, and its lengths"""
    B, Sq, Sk, nh, nkv, causal, kl, heads = case
    r = rng(B + Sq + hd)
    ql = None
    if isinstance(kl, str):
        lens = [int(t) for t in r.integers(Sk // 4, Sk + 1, B)]
        if kl == "some empty":
            lens[3], lens[B - 5], lens[B - 1] = 0, 1, 0
            ql = [int(t) for t in r.integers(0, Sq + 1, B)]
        kl = lens
    q = enc(0.5 * r.standard_normal((B, Sq, 2 * nh * hd)), dt)
    k = enc(r.standard_normal((B, Sk, 2 * nkv * hd)), dt)
    j = np.arange(Sk)
    v = np.zeros((Sk, 2 * hd), np.float32)
    v[j, j // block_of(Sk) % (2 * hd)] = 16.0
    v = np.ascontiguousarray(np.broadcast_to(np.tile(enc(v, dt), nkv), (B, Sk, 2 * nkv * hd)))
    lam = np.zeros((1, 4, hd), np.float32)
    lam[0, 2:] = np.sqrt(np.log(1.0 - LAMBDA) / hd)
    return q, k, v, lam, ql, kl


CASES = [c + t for c in CUTS + MORE for t in ((F16, 64, True), (BF16, 32, False))]
NAMES = "B,Sq,Sk,nh,nkv,causal,kl,heads,dt,hd,norm"


@pytest.mark.parametrize(NAMES, CASES)
def test_a_lost_block_shows(B, Sq, Sk, nh, nkv, causal, kl, heads, dt, hd, norm):
    q, k, v, lam, ql, lens = cut_case((B, Sq, Sk, nh, nkv, causal, kl, heads), hd, dt)
    lens = [Sk] * B if lens is None else lens
    b = max((b for b in range(B) if ql is None or ql[b]), key=lambda b: lens[b])   # the longest: a block weighs least
    row = (Sq if ql is None else ql[b]) - 1                                        # the last row sees all keys
    w = np.ones(2 * hd) if norm else None

    def one(keys):
        o, t, _ = attn_ref(dec(q[b:b + 1, row:row + 1, :2 * hd], dt), dec(k[b:b + 1, keys, :2 * hd], dt), dec(v[b:b + 1, keys, :2 * hd], dt),
                           lam.astype(np.float64), w, [1], [len(keys)], False, np.float64(np.float32(hd ** -0.5)), 0.0, 1e-5, 1, 1, hd, dt)
        return o, t

    keys = np.arange(lens[b])
    want, tol = one(keys)
    block = block_of(Sk)
    blocks = lens[b] // block
    r = rng(blocks)
    for i in {0, blocks - 1, *(int(t) for t in r.integers(0, blocks, 4))}:
        at = np.s_[i * block:(i + 1) * block]
        for changed in (np.delete(keys, at), np.concatenate([keys, keys[at]])):
            assert (np.abs(one(changed)[0] - want) / tol).max() > 2.0, i   # the answer itself is within one


@pytest.mark.gpu
@pytest.mark.parametrize(NAMES, CASES)
def test_no_block_is_lost(tsn, rt, B, Sq, Sk, nh, nkv, causal, kl, heads, dt, hd, norm):
    q, k, v, lam, ql, lens = cut_case((B, Sq, Sk, nh, nkv, causal, kl, heads), hd, dt)
    w = np.ones(2 * hd, np.float32) if norm else None
    out = np.full(q.shape, SENTINEL[dt], NP[dt])
    qb, kb, vb, lb, ob = (rt.array(t) for t in (q, k, v, lam, out))
    wb, qlb, klb = (None if t is None else rt.array(np.asarray(t, f)) for t, f in ((w, np.float32), (ql, np.int32), (lens, np.int32)))
    rt.diff_attention(tsn.diff_attn_spec(dt, B, Sq, Sk, nh, nkv, hd, causal=causal, lambda_init=0.0), qb, kb, vb, lb, wb, qlb, klb, ob)
    rt.sync()
    got = ob.numpy()
    want, tol, live = attn_ref(dec(q, dt), dec(k, dt), dec(v, dt), lam.astype(np.float64), None if w is None else w.astype(np.float64),
                               [Sq] * B if ql is None else ql, [Sk] * B if lens is None else lens, causal,
                               np.float64(np.float32(hd ** -0.5)), 0.0, np.float64(np.float32(1e-5)), nh, nkv, hd, dt, heads)
    check(dec(got, dt)[live], want[live], tol[live])
    for t in (qb, kb, vb, lb, ob, wb, qlb, klb):
        if t is not None:
            t.free()
