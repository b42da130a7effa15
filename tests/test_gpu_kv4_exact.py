"""Attention over the 4-bit KV cache where rounding to fp16's range could cost more than fp32's precision: positions far below
a sink, against float64 sums of what each row is made of."""
import numpy as np
import pytest

import kv4_ref as R
from test_gpu_kv4 import Cache, append, attend

pytestmark = pytest.mark.gpu

# heads, KV heads, head size, rows of the run: rows by themselves; one block of 128 queries, two and more (pairs); the runs of
# the other head sizes
SHAPES = [(8, 2, 64, 1), (4, 2, 96, 1), (8, 1, 128, 1), (4, 1, 256, 1), (4, 1, 64, 24), (4, 1, 128, 24), (8, 1, 64, 40), (16, 2, 128, 300),
          (4, 2, 96, 24), (2, 1, 256, 24)]


def held(wl, k, v):
    """A cache of the keys and values [n][kv_heads][hd] (float64 or float32), and what it holds of them."""
    n, kv_heads, hd = k.shape
    c = Cache(1, kv_heads, hd, n)
    k, v = (np.ascontiguousarray(x, dtype=np.float32) for x in (k, v))
    append(wl, c, [0] * n, range(n), k, k, v, np.zeros((1, 1, 2), np.float32), 0, False)
    raw = c.host()[0]
    return c, *(R.read(raw, kv_heads, hd, n, e) for e in (False, True))


def by_terms(q, k, v, p, scale):
    """One row over positions 0 .. p: (out, bound) in float64, the bound from the sizes of the sums' terms.

    Keys and values are held exactly. A query's element is off by 2^-22 of itself (two fp16 roundings, 2^-11 each) and three
    half steps of 2^-24 (its scale), with an absolute floor of 2^-38 of the row's largest; the dropped product of remainders is
    2^-22 of a term: below 2^-20 of sum |q_i k_i| together. A score's fp32 sums have at most 3 hd / 16 MMA steps and 8 more
    additions, each cut off at 2^-23 of the terms so far; where one product is not zero they are exact. The exponential's
    argument is rounded at 2^-24 of at most 64 and the exponential is off by 2^-22: 2^-17 together. So a weight has a factor
    exp(delta), delta = (2^-20 + (3 hd / 16 + 8) 2^-23 [several terms]) sum |q_i k_i| scale + 2^-17, and the row's sum too.
    Weights are split as queries are (2^-20), and the sums over n positions have at most 40 + n / 64 steps of 2^-23 in a
    row, the row's sum of weights too: all these relative to sum w_j |v_j|. What is left below fp16's range: 2^-39 of a step's largest
    weight for each of its 128 positions, or, for rows by themselves, 2^-41 max(1, the largest scale) a position."""
    heads, hd = q.shape
    g, n = heads // k.shape[1], p + 1
    out, bound = np.zeros((heads, hd)), np.zeros((heads, hd))
    for h in range(heads):
        kk, vv, qq = k[:n, h // g], v[:n, h // g], np.asarray(q[h], np.float64)
        s = kk @ qq * scale
        w = np.exp(s - s.max())
        w /= w.sum()
        out[h] = w @ vv
        terms = np.abs(kk * qq)
        size = (terms.sum(1) + 2.0 ** -38 * np.abs(qq).max() * np.abs(kk).sum(1)) * abs(scale)
        several = (terms > 0).sum(1) > 1
        delta = ((2.0 ** -20 + several * (3 * hd / 16 + 8) * 2.0 ** -23) * size).max() + 2.0 ** -17
        rel = 2 * delta * (1 + delta) + 2.0 ** -20 + 2 * (40 + n / 64) * 2.0 ** -23
        top = np.abs(vv).max()
        floor = max(min(n, 128) * 2.0 ** -39 * top, n * 2.0 ** -41 * max(1.0, top / 8))
        bound[h] = rel * (w @ np.abs(vv)) + w.max() * floor
    return out, bound


@pytest.mark.parametrize("heads,kv_heads,hd,rows", SHAPES)
@pytest.mark.parametrize("nats", [8, 12, 15, 18])
@pytest.mark.parametrize("vscale", [1.0, 0.01])
def test_weights_far_below_a_sink_keep_their_precision(wl, heads, kv_heads, hd, rows, nats, vscale):
    """The first position takes nearly all of the weight and has a value of zero: the output is what the others, far below it,
    sum to."""
    rng = np.random.default_rng(heads * hd + rows + nats)
    n, scale = 4000, hd ** -0.5
    k, v = (rng.standard_normal((n, kv_heads, hd)) for _ in range(2))
    k[0], v[0], k[:, :, 0] = 0, 0, 0
    k[0, :, 0] = -8.0                                   # (its block's scale is 1: held exactly)
    c, hk, hv = held(wl, k, v * vscale)
    q = (rng.standard_normal((rows, heads, hd)) * 0.3).astype(np.float32)
    q[:, :, 0] = -nats / 8 / scale
    pos = list(range(n - rows, n))
    out = attend(wl, c, [0] * rows, pos, q, runs=rows)
    for t in list(range(0, rows, 23)) + [rows - 1]:
        want, bound = by_terms(q[t], hk, hv, pos[t], scale)
        off = np.abs(out[t] - want)
        assert (off <= bound).all(), (t, float((off / bound).max()), float(off.max() / np.abs(want).max()))
    assert wl.lib().wl_kernel_status(0) == 0


@pytest.mark.parametrize("heads,kv_heads,hd,rows", SHAPES)
@pytest.mark.parametrize("kscale", [1e-6, 1e-5, 2e-4, 1e-3, 1e5])
def test_keys_of_any_scale(wl, heads, kv_heads, hd, rows, kscale):
    """Keys whose scales are subnormal in fp16, or near its largest value, under queries that are large or small in return."""
    rng = np.random.default_rng(heads * hd + rows)
    n, scale = 700, hd ** -0.5
    k, v = (rng.standard_normal((n, kv_heads, hd)) for _ in range(2))
    c, hk, hv = held(wl, k * kscale, v)
    q = (rng.standard_normal((rows, heads, hd)) * 2 / kscale).astype(np.float32)
    pos = list(range(n - rows, n))
    out = attend(wl, c, [0] * rows, pos, q, runs=rows)
    for t in list(range(0, rows, 23)) + [rows - 1]:
        want, bound = by_terms(q[t], hk, hv, pos[t], scale)
        off = np.abs(out[t] - want)
        assert (off <= bound).all(), (t, float((off / bound).max()))
    assert wl.lib().wl_kernel_status(0) == 0


@pytest.mark.parametrize("heads,kv_heads,hd,rows", SHAPES)
def test_steps_with_keys_of_two_scales(wl, heads, kv_heads, hd, rows):
    """Keys of 60000 and more among small ones, in steps of their own and beside them: the small ones keep what 2^-24 of a
    step's largest key scale leaves them."""
    rng = np.random.default_rng(heads * hd + rows)
    n, scale = 700, hd ** -0.5
    k, v = (rng.standard_normal((n, kv_heads, hd)) for _ in range(2))
    k *= 0.05
    big = [130, 131, 300, 690]
    k[:, :, 0] = 0
    k[big] = 0
    k[big, :, 0] = -8.0 * 10240                         # (scales of 10240: held exactly)
    c, hk, hv = held(wl, k, v)
    q = rng.standard_normal((rows, heads, hd)).astype(np.float32)
    q[:, :, 0] = 1e-4
    q[:, ::2, 0] = -1e-4
    pos = list(range(n - rows, n))
    out = attend(wl, c, [0] * rows, pos, q, runs=rows)
    for t in list(range(0, rows, 23)) + [rows - 1]:
        want, bound = by_terms(q[t], hk, hv, pos[t], scale)
        off = np.abs(out[t] - want)
        assert (off <= bound).all(), (t, float((off / bound).max()))


@pytest.mark.parametrize("heads,kv_heads,hd,rows", SHAPES)
@pytest.mark.parametrize("size", [1e8, 1e9, 8e9, 1e33, 1e36, 3e38])
def test_queries_of_any_finite_size(wl, heads, kv_heads, hd, rows, size):
    """Finite scores of finite queries, up to the largest floats: one position has a key where the queries are that large, and takes
    all of the weight."""
    rng = np.random.default_rng(hd + rows)
    n, scale, kv = 60, hd ** -0.5, 2.0 ** -6
    k, v = np.zeros((n, kv_heads, hd)), rng.standard_normal((n, kv_heads, hd))
    k[7, :, 3] = -8 * kv
    c, hk, hv = held(wl, k, v)
    q = np.zeros((rows, heads, hd), np.float32)
    q[:, :, 3] = -size
    pos = list(range(n - rows, n)) if rows <= 40 else [n - 1] * rows
    out = attend(wl, c, [0] * rows, pos, q, runs=rows)
    # a weight of 1 times an exact value, divided by the sum 1: a few roundings of 2^-22
    want = np.repeat(hv[7], heads // kv_heads, 0)
    assert (np.abs(out - want) <= 2.0 ** -20 * np.abs(want)).all()
