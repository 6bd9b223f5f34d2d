"""The block operators where rounding, range and the cuts of the work could lose something that evenly spread inputs do
not show. References, tolerances and the call itself are those of test_gpu_blockops."""
import numpy as np
import pytest

from test_gpu_blockops import BF16, F16, attn_case

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- one key far above the others

@pytest.mark.parametrize("dt,hd", [(F16, 64), (F16, 32), (BF16, 64)])
@pytest.mark.parametrize("nats", [10.0, 12.4, 14.2, 15.2])
@pytest.mark.parametrize("at", ["first", "middle", "last"])
@pytest.mark.parametrize("B,Sq,Sk,nh,heads", [
    (2, 397, 397, 8, (0, 7)),          # few-row tiles of a workgroup each
    (1, 1300, 3000, 50, (0, 49)),      # wide tiles
    (1, 5, 20000, 2, None),            # keys shared out
])
def test_diff_attention_one_key_above(tsn, rt, dt, hd, nats, at, B, Sq, Sk, nh, heads):
    """One key that every row prefers by 10 to 15 nats, with a value of zeros, and equal others that make up the
    result: their probabilities of 2^-14.4 to 2^-22 of the largest are all rounded alike, so that a rounding step larger than the
    type's own (f16 has steps of 2^-24 below 2^-14) shows as it is. The tolerance is the one of any other input."""
    def make(r, q, k, v):
        j = {"first": 0, "middle": Sk // 2 + 1, "last": Sk - 1}[at]
        q[:], k[:] = 1.0, 0.0
        k[:, j] = nats / np.sqrt(hd)
        v[:] = 50.0 * (1.0 + np.abs(v))
        v[:, j] = 0.0
        return q, k, v

    attn_case(tsn, rt, dt, B, Sq, Sk, nh, nh, hd, make=make, norm=False, heads=heads)


# ---------------------------------------------------------------- values whose squares leave f32

@pytest.mark.parametrize("hd", [64, 32])
@pytest.mark.parametrize("Sq,Sk,nh,heads,pad", [
    (40, 300, 4, None, 0), (1300, 1400, 50, (0, 49), 0), (1, 9000, 2, None, 0), (9, 300, 2, None, 1)])
def test_diff_attention_small_values(tsn, rt, hd, Sq, Sk, nh, heads, pad):
    """bf16 values of 2^-80 under the norm: their squares are zeros in f32, what is left of the mean square is eps
    (2^-160 beside 1e-5), so that rows are scaled by 1/sqrt(eps) and not lost"""
    def make(r, q, k, v):
        return q, k, v * 2.0 ** -80

    attn_case(tsn, rt, BF16, 1, Sq, Sk, nh, nh, hd, make=make, heads=heads, pad=(pad,) * 4)


# ---------------------------------------------------------------- scores far from one

@pytest.mark.parametrize("hd", [64, 32])
@pytest.mark.parametrize("scale", [0.0, 2.0 ** -112])
@pytest.mark.parametrize("Sq,Sk,nh,heads,pad", [
    (40, 300, 4, None, 0), (1300, 1400, 50, (0, 49), 0), (1, 9000, 2, None, 0), (9, 300, 2, None, 1)])
def test_diff_attention_large_products(tsn, rt, hd, scale, Sq, Sk, nh, heads, pad):
    """bf16 q and k of 2^55: products of up to 2^120, which a scale of 0 turns into equal weights and one of 2^-112 into
    scores of a few units"""
    attn_case(tsn, rt, BF16, 1, Sq, Sk, nh, nh, hd, True, make=lambda r, q, k, v: (q * 2.0 ** 55, k * 2.0 ** 55, v),
              heads=heads, pad=(pad,) * 4, scale=scale)


# ---------------------------------------------------------------- rows that are not whole 16-byte chunks

@pytest.mark.parametrize("hd", [64, 32])
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("B,Sq,Sk,nh,nkv,causal,ql,kl,shared_lambda", [
    (2, 34, 200, 4, 2, False, None, None, True),
    (3, 40, 130, 4, 4, False, [40, 0, 7], [130, 64, 0], False),
    (3, 70, 70, 6, 2, True, [70, 33, 1], [70, 33, 1], False),
    (2, 1, 1000, 4, 1, True, None, [1000, 999], False),
    (2, 33, 65, 2, 2, True, [33, 20], [20, 65], True),       # rows before the first key
    (1, 1, 1, 1, 1, False, None, None, True),
])
def test_diff_attention_odd_places(tsn, rt, dt, hd, norm, B, Sq, Sk, nh, nkv, causal, ql, kl, shared_lambda):
    """odd strides and columns: the kernel that reads element by element, in each of its widths and types, under every mask,
    with and without its norm"""
    attn_case(tsn, rt, dt, B, Sq, Sk, nh, nkv, hd, causal, ql, kl, lam_heads=1 if shared_lambda else nh, norm=norm,
              junk=np.nan, pad=(1, 3, 5, 7), col=1)


# ---------------------------------------------------------------- values far above one

@pytest.mark.parametrize("hd", [64, 32])
@pytest.mark.parametrize("Sq,Sk,nh,heads,pad", [
    (40, 300, 4, None, 0), (1300, 1400, 50, (0, 49), 0), (1, 9000, 2, None, 0), (9, 300, 2, None, 1)])
def test_diff_attention_large_values(tsn, rt, hd, Sq, Sk, nh, heads, pad):
    """bf16 values of up to 2^57 under the norm (their squares add up to less than 2^128), of up to 2^113 without it"""
    for power, norm in ((55, True), (111, False)):
        attn_case(tsn, rt, BF16, 1, Sq, Sk, nh, nh, hd, heads=heads, make=lambda r, q, k, v: (q, k, np.clip(v, -4, 4) * 2.0 ** power),
                  pad=(pad,) * 4, norm=norm)
