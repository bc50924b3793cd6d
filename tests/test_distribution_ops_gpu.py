"""Operators on a model's distribution against their definitions in 64 bits:
cngpt_cuda_sample, cngpt_cuda_topk, cngpt_cuda_distill.

Tokens and indices are whole numbers and have to be equal. Floating results
are held to bounds that count roundings of half a step, 2^-24 relative.
"""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from cngpt_b200 import abi

pytestmark = pytest.mark.gpu
EPS = float(torch.finfo(torch.float32).eps) / 2  # one rounding of an fp32 result
INF = math.inf
NAN = math.nan


def dev(a, dtype=None):
    return None if a is None else torch.as_tensor(np.ascontiguousarray(a), dtype=dtype).cuda()


def ptr(t):
    return None if t is None else t.data_ptr()


def padded(x, ld, shift=0, fill=NAN):
    """x [rows, V] on the device with row pitch ld, `shift` floats behind an
    aligned address, surrounded by `fill`; returns (buffer, pointer)."""
    rows, V = x.shape
    buf = torch.full((shift + rows * ld + 8,), fill, dtype=torch.float32, device="cuda")
    view = buf[shift:shift + rows * ld].view(rows, ld)
    view[:, :V] = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    return buf, buf.data_ptr() + 4 * shift


# ------------------------------------------------------------------ sample
def ref_sample(x, T, k, p, mp, u):
    """(token, logprob) of one row from the definition, in 64 bits."""
    x = np.asarray(x, np.float64)
    c = np.flatnonzero(x > -INF)  # NaN and -inf are never drawn
    if c.size == 0:
        return -1, -INF
    c = c[np.argsort(-x[c], kind="stable")]
    if not T > 0 or p <= 0:
        return int(c[0]), 0.0
    mx = x[c[0]]
    if mx == INF:
        w = (x[c] == INF).astype(np.float64)
    else:
        with np.errstate(over="ignore"):
            w = np.exp((x[c] - mx) / T)
    if k > 0:
        c, w = c[:k], w[:k]
    if p < 1:
        before = np.cumsum(w) - w
        n = max(1, int(np.sum(before < p * w.sum())))
        c, w = c[:n], w[:n]
    if mp > 0:
        n = int(np.sum(w >= min(1.0, mp)))
        c, w = c[:n], w[:n]
    o = np.argsort(c)
    c, w = c[o], w[o]
    c, w = c[w > 0], w[w > 0]
    cum = np.cumsum(w)
    at = min(int(np.searchsorted(cum, u * cum[-1], side="right")), len(c) - 1)
    return int(c[at]), math.log(w[at]) - math.log(cum[-1])


def check_sample(lib, x, T=None, k=None, p=None, mp=None, u=None, ld=None, shift=0):
    rows, V = x.shape
    ld = ld or V
    buf, at = padded(x, ld, shift, fill=INF)
    arr = lambda a, t: None if a is None else np.asarray(a, t)  # noqa: E731
    T, k, p, mp, u = arr(T, np.float32), arr(k, np.int32), arr(p, np.float32), arr(mp, np.float32), arr(u, np.float32)
    dT, dk, dp, dm, du = dev(T), dev(k), dev(p), dev(mp), dev(u)
    tok = torch.full((rows + 1,), -77, dtype=torch.int32, device="cuda")
    lp = torch.full((rows + 1,), 77.0, dtype=torch.float32, device="cuda")
    abi.check(lib, lib.cngpt_cuda_sample(at, ld, rows, V, ptr(dT), ptr(dk), ptr(dp), ptr(dm), ptr(du), ptr(tok),
                                         ptr(lp)), "sample")
    abi.check(lib, lib.cngpt_cuda_check(), "sync")
    got, glp = tok.cpu().numpy(), lp.cpu().numpy()
    assert got[rows] == -77 and glp[rows] == 77.0  # nothing written behind the last row
    one = lambda a, r, d: d if a is None else float(a[r])  # noqa: E731
    for r in range(rows):
        t, l = ref_sample(x[r], one(T, r, 1.0), int(one(k, r, 0)), one(p, r, 1.0), one(mp, r, 0.0), float(u[r]))
        assert got[r] == t, (r, got[r], t)
        # the log is rounded once; the weights' sum is held to about 1e-9
        assert glp[r] == l or abs(float(glp[r]) - l) <= EPS * abs(l) + 1e-8, (r, glp[r], l)  # in 64 bits
    return got[:rows]


def logits(rows, V, seed, spread=2.0):
    g = np.random.default_rng(seed)
    x = g.standard_normal((rows, V)) * spread
    x[g.random((rows, V)) < 0.02] += 6.0
    return x.astype(np.float32)


@pytest.mark.parametrize("V", [1, 2, 31, 50257, 65, 1000, 4097, 128256])
@pytest.mark.parametrize("mode", ["plain", "topk", "topp", "minp", "all"])
def test_sample_sizes_and_filters(lib, cuda, V, mode):
    rows = 7 if V > 5000 else 33
    g = np.random.default_rng(V)
    kw = dict(T=g.uniform(0.3, 2.0, rows), u=g.random(rows))
    if mode in ("topk", "all"):
        kw["k"] = g.integers(1, max(2, min(V, 3000)), rows)
    if mode in ("topp", "all"):
        kw["p"] = g.uniform(0.05, 0.999, rows)
    if mode in ("minp", "all"):
        kw["mp"] = g.uniform(0.0, 0.5, rows)
    check_sample(lib, logits(rows, V, V + 1), **kw)


@pytest.mark.parametrize("rows", [1, 2, 40, 149, 300])
def test_sample_row_counts(lib, cuda, rows):
    g = np.random.default_rng(rows)
    check_sample(lib, logits(rows, 50257, rows), T=g.uniform(0.5, 1.5, rows), k=g.integers(-1, 100, rows),
                 p=g.uniform(0.5, 1.2, rows), mp=g.uniform(-0.1, 0.2, rows), u=g.random(rows))


@pytest.mark.parametrize("ld,shift", [(1003, 0), (1003, 1), (1004, 3), (2048, 2)])
def test_sample_strides_and_alignment(lib, cuda, ld, shift):
    g = np.random.default_rng(3)
    check_sample(lib, logits(9, 1003, 5), T=np.full(9, 0.9), k=np.full(9, 40), p=np.full(9, 0.9), u=g.random(9), ld=ld,
                 shift=shift)


@pytest.mark.parametrize("V", [64, 5000, 50257])
def test_sample_ties_go_to_the_lowest_index(lib, cuda, V):
    """Few distinct values, so that every threshold falls inside a run of equals."""
    g = np.random.default_rng(V)
    rows = 24
    x = g.integers(-3, 3, (rows, V)).astype(np.float32)
    x[0] = 0.0
    x[1] = -0.0
    x[2, ::2] = -0.0
    check_sample(lib, x, T=g.uniform(0.5, 2.0, rows), k=g.integers(1, V, rows), p=g.uniform(0.1, 0.99, rows),
                 u=g.random(rows))
    check_sample(lib, x, k=g.integers(1, V, rows), u=g.random(rows))
    check_sample(lib, x, p=g.uniform(0.1, 0.99, rows), u=g.random(rows))


def test_sample_borders_of_equal_weights(lib, cuda):
    """Equal weights: every border is exact, a number on it takes the next token."""
    x = np.zeros((8, 8), np.float32)
    u = np.arange(8) / 8
    assert check_sample(lib, x, u=u).tolist() == list(range(8))
    got = check_sample(lib, x, p=np.full(8, 0.5), u=u)
    assert got.max() == 3 and got.min() == 0


def test_sample_parameter_limits(lib, cuda):
    rows = 32
    x = logits(rows, 777, 9)
    u = np.random.default_rng(1).random(rows)
    one = lambda *v: np.resize(np.array(v, np.float64), rows)  # noqa: E731
    tiny = float(np.float32(1e-45))
    check_sample(lib, x, T=one(0.0, -1.0, NAN, tiny, INF, 1e30, 1e-3, 100.0), u=u)
    check_sample(lib, x, k=one(0, -5, 1, 776, 777, 778, 2**31 - 1, 2).astype(np.int64), u=u)
    check_sample(lib, x, p=one(0.0, -1.0, tiny, 1.0, 2.0, 0.99999994, 1e-7, INF), u=u)
    check_sample(lib, x, mp=one(0.0, -1.0, 1.0, 2.0, tiny, 0.5, INF, 0.999), u=u)
    check_sample(lib, x, T=one(0.7), u=one(0.0, 0.99999994, 0.5, tiny))
    check_sample(lib, x, T=one(0.02), u=one(0.0, 0.99999994, 0.5, tiny))
    nan = check_sample(lib, x, p=one(NAN), mp=one(NAN), u=u)  # NaN switches a filter off
    assert (nan == check_sample(lib, x, u=u)).all()


@pytest.mark.parametrize("V", [40, 50257])
def test_sample_infinities_nan_and_empty_rows(lib, cuda, V):
    g = np.random.default_rng(2)
    x = logits(16, V, 3)
    x[0] = -INF
    x[1] = NAN
    x[2, :] = -INF
    x[2, V - 1] = -2.0
    x[3, g.random(V) < 0.9] = -INF
    x[4, g.random(V) < 0.5] = NAN
    x[5, [3, 7, 30]] = INF
    x[6, 0] = INF
    x[7] = -3.4028235e38
    x[7, 5] = 3.4028235e38
    x[8] = -3.4028235e38
    x[9, 1:] = -INF
    x[10, ::2] = -INF
    x[10, 1::2] = NAN
    x[11, 2] = 3e38
    for kw in (dict(), dict(k=np.full(16, 5)), dict(p=np.full(16, 0.9)), dict(mp=np.full(16, 0.1)),
               dict(k=np.full(16, V // 2), p=np.full(16, 0.95), mp=np.full(16, 0.001)), dict(T=np.zeros(16))):
        check_sample(lib, x, u=g.random(16), **kw)


def test_sample_flat_rows_keep_most_of_the_vocabulary(lib, cuda):
    """Thresholds that fall into the body of a flat distribution."""
    g = np.random.default_rng(5)
    x = (g.standard_normal((12, 50257)) * 0.05).astype(np.float32)
    x[6:] = g.random((6, 50257), np.float32) * 1e-6 + 4.0
    check_sample(lib, x, p=g.uniform(0.3, 0.99, 12), u=g.random(12))
    check_sample(lib, x, k=g.integers(10000, 50000, 12), u=g.random(12))
    check_sample(lib, x, k=g.integers(10000, 50000, 12), p=g.uniform(0.3, 0.99, 12), u=g.random(12))


@pytest.mark.parametrize("V", [513, 2000, 20011, 50257, 262144])
@pytest.mark.parametrize("rows", [1, 24])
def test_sample_nuclei_from_one_token_to_all(lib, cuda, rows, V):
    """top-p over rows whose nucleus is a few tokens, some hundreds, thousands, or
    cut out of a run of equal logits, with the whole mass in any part of the row."""
    g = np.random.default_rng(V + rows)
    base = logits(8, V, V, spread=1.0)
    base[1] *= 8.0                                   # a few tokens
    base[2] = np.float32(0.01) * base[2]             # nearly flat
    base[3, g.permutation(V)[:600]] = 9.0            # a run of equal ones around the border
    base[4, : V - 400] = -INF                        # all in the last stretch
    base[5, g.random(V) < 0.97] = -INF
    base[6] = np.where(g.random(V) < 0.5, np.float32(1.0), np.float32(0.0))  # two values
    base[7, 5] = 60.0                                # one token outweighs the others
    x = base[np.arange(rows) % 8] if rows > 1 else base[3:4]
    p = g.choice([0.05, 0.3, 0.6, 0.9, 0.97, 0.9999], rows)
    check_sample(lib, x, T=g.choice([0.01, 0.4, 1.0, 30.0], rows), p=p, u=g.random(rows))
    check_sample(lib, x, T=g.choice([0.7, 1.0], rows), p=p, mp=g.uniform(0.0, 0.3, rows), u=g.random(rows))
    check_sample(lib, x, k=np.full(rows, min(V, 700)), p=p, u=g.random(rows))
    check_sample(lib, x, k=np.full(rows, 200), p=p, mp=np.full(rows, 0.01), u=g.random(rows))


def test_sample_without_logprob_and_repeatable(lib, cuda):
    x = torch.from_numpy(logits(50, 50257, 8)).cuda()
    u = torch.rand(50, device="cuda")
    got = []
    for _ in range(3):
        tok = torch.empty(50, dtype=torch.int32, device="cuda")
        abi.check(lib, lib.cngpt_cuda_sample(ptr(x), 50257, 50, 50257, None, None, None, None, ptr(u), ptr(tok), None))
        abi.check(lib, lib.cngpt_cuda_check())
        got.append(tok.cpu())
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


# -------------------------------------------------------------------- topk
def ref_topk(x, k):
    key = np.where(np.isnan(x), -INF, x)
    o = np.lexsort((np.arange(x.shape[1])[None, :].repeat(x.shape[0], 0), np.isnan(x), -key), axis=1)[:, :k]
    return np.take_along_axis(x, o, 1), o


def check_topk(lib, x, k, ld=None, shift=0):
    rows, V = x.shape
    ld = ld or V
    buf, at = padded(x, ld, shift, fill=INF)
    val = torch.full((rows * k + 3,), 77.0, device="cuda")
    idx = torch.full((rows * k + 3,), -77, dtype=torch.int32, device="cuda")
    abi.check(lib, lib.cngpt_cuda_topk(at, ld, rows, V, k, ptr(val), ptr(idx)), "topk")
    abi.check(lib, lib.cngpt_cuda_check(), "sync")
    v, i = val.cpu().numpy(), idx.cpu().numpy()
    assert (v[rows * k:] == 77.0).all() and (i[rows * k:] == -77).all()
    rv, ri = ref_topk(x, k)
    assert np.array_equal(i[: rows * k].reshape(rows, k), ri)
    assert np.array_equal(v[: rows * k].reshape(rows, k), rv, equal_nan=True)


@pytest.mark.parametrize("V,k", [(1, 1), (5, 5), (31, 3), (65, 64), (1000, 1), (1024, 1024), (4099, 100), (32003, 20),
                                 (50257, 1), (50257, 64), (50257, 257), (50257, 1024), (128256, 128)])
@pytest.mark.parametrize("rows", [1, 37])
def test_topk_sizes(lib, cuda, V, k, rows):
    check_topk(lib, logits(rows, V, V + k), k)


@pytest.mark.parametrize("ld,shift", [(5003, 0), (5003, 1), (5003, 2), (5004, 3), (8192, 1)])
def test_topk_strides_and_alignment(lib, cuda, ld, shift):
    check_topk(lib, logits(6, 5003, 4), 50, ld, shift)


@pytest.mark.parametrize("k", [1, 40, 500, 1024])
def test_topk_ties_orders_and_special_values(lib, cuda, k):
    g = np.random.default_rng(k)
    V = 50257
    x = logits(13, V, 6)
    x[0] = g.integers(-3, 3, V)
    x[1] = 0.0
    x[2] = np.arange(V)  # rising: every element is a new maximum
    x[3] = -np.arange(V)
    x[4] = -INF
    x[5] = NAN
    x[6, g.random(V) < 0.5] = -INF
    x[7, g.random(V) < 0.5] = NAN
    x[8] = -INF
    x[8, 100:120] = 1.0
    x[8, 200:230] = NAN
    x[9, g.integers(0, V, 30)] = INF
    x[10, ::3] = 9.0
    x[11] = np.where(np.arange(V) % 2, 0.0, -0.0)
    x[12] = np.sort(x[12])[::-1]
    check_topk(lib, x, k)


@pytest.mark.parametrize("tail", [0, 1, 3])
def test_topk_numbers_after_nan(lib, cuda, tail):
    """Rows of NaN with as many numbers as are asked for, and larger ones at the
    very end: whatever was cut before must let those pass."""
    V = 4096 + 100 + tail
    x = np.full((3, V), NAN, np.float32)
    x[:, [3, 700, 1500, 2222, 4000]] = [1.0, -2.0, 3.0, -INF, 5.0]
    x[:, [4100, 4120, 4130, 4140, 4150]] = [0.5, -INF, 2.0, -3.0, 4.0]
    if tail:
        x[1, V - tail:] = 100.0 + np.arange(tail)
        x[2, V - 1] = -INF
    check_topk(lib, x, 10)
    check_topk(lib, x, 9)
    check_topk(lib, x, 12)


def test_topk_many_rows(lib, cuda):
    check_topk(lib, logits(700, 3001, 11), 33)


@pytest.mark.parametrize("rows,V,k", [(1783, 7, 7), (1783, 130, 128), (1783, 512, 100), (1779, 513, 128), (1783, 1300, 24),
                                      (1778, 4096, 128), (1778, 4096, 1), (30, 400, 60), (1778, 4095, 129)])
@pytest.mark.parametrize("shift", [0, 3])
def test_topk_many_short_rows(lib, cuda, rows, V, k, shift):
    g = np.random.default_rng(V + k)
    x = logits(rows, V, V)
    x[0] = g.integers(-3, 3, V)
    x[1] = 0.0
    x[2] = np.arange(V)
    x[3] = -np.arange(V)
    x[4], x[5] = -INF, NAN
    x[6, g.random(V) < 0.9], x[7, g.random(V) < 0.9] = -INF, NAN
    x[8, V // 3:], x[9, : V // 2] = NAN, -INF
    x[10, g.integers(0, V, 3)] = INF
    x[11] = np.where(np.arange(V) % 2, 0.0, -0.0)
    x[12, : V - 1] = NAN
    x[rows - 1] = np.sort(x[rows - 1])
    check_topk(lib, x, k, V + shift, shift)


# ------------------------------------------------------------------ distill
def ref_distill(x, tv, ti, tgt, tau, alpha, scale):
    """(loss, row_loss, dlogits, gradient's terms in size, largest |x - max|)."""
    x = np.asarray(x, np.float64)
    rows, V = x.shape
    tau, alpha, scale = float(np.float32(tau)), float(np.float32(alpha)), float(np.float32(scale))
    row, grad, size = np.zeros(rows), np.zeros((rows, V)), np.zeros((rows, V))
    for r in range(rows):
        m = x[r].max()
        if m == -INF:
            continue
        with np.errstate(divide="ignore", invalid="ignore"):
            lt = (x[r] - m) / tau
            lt = lt - math.log(np.exp(lt).sum())
            l1 = x[r] - m
            l1 = l1 - math.log(np.exp(l1).sum())
        if tv is not None and alpha > 0:
            ok = [(int(i), float(v)) for i, v in zip(ti[r], tv[r]) if 0 <= i < V and v > -INF]
            if ok:
                i = np.array([a for a, _ in ok])
                z = np.array([b for _, b in ok], np.float64) / tau
                lp = z - z.max()
                lp = lp - math.log(np.exp(lp).sum())
                p = np.exp(lp)
                use = p > 0
                row[r] += alpha * tau * tau * np.sum(p[use] * (lp[use] - lt[i][use]))
                grad[r] += alpha * tau * np.exp(lt)
                size[r] += alpha * tau * np.exp(lt)
                np.add.at(grad[r], i, -alpha * tau * p)
                np.add.at(size[r], i, alpha * tau * p)
        if tgt is not None and alpha < 1 and 0 <= tgt[r] < V:
            row[r] -= (1 - alpha) * l1[tgt[r]]
            grad[r] += (1 - alpha) * np.exp(l1)
            size[r] += (1 - alpha) * np.exp(l1)
            grad[r, tgt[r]] -= 1 - alpha
            size[r, tgt[r]] += 1 - alpha
    return scale * row.sum(), row, scale * grad, abs(scale) * size


def run_distill(lib, x, tv, ti, tgt, tau, alpha, scale, grad=True, inplace=False, ld=None, shift=0, ldd=None):
    rows, V = x.shape
    ld = ld or V
    k = 0 if tv is None else tv.shape[1]
    buf, at = padded(x, ld, shift, fill=5.0)
    dtv, dti, dtg = dev(tv), dev(ti), dev(tgt)
    loss = torch.full((2,), 77.0, device="cuda")
    row = torch.full((rows + 1,), 77.0, device="cuda")
    d, dat = None, None
    if grad:
        ldd = ld if inplace else ldd or V
        d, dat = (buf, at) if inplace else padded(np.zeros((rows, V), np.float32), ldd, shift, fill=5.0)
    abi.check(lib, lib.cngpt_cuda_distill(at, ld, rows, V, ptr(dtv), ptr(dti), k, ptr(dtg), tau, alpha, scale, ptr(loss),
                                          ptr(row), dat, ldd or 0), "distill")
    abi.check(lib, lib.cngpt_cuda_check(), "sync")
    loss, row = loss.cpu().numpy(), row.cpu().numpy()
    assert loss[1] == 77.0 and row[rows] == 77.0
    g = None
    if grad:
        full = d.cpu().numpy()
        assert (full[:shift] == 5.0).all() and (full[shift + rows * ldd:] == 5.0).all()
        full = full[shift:shift + rows * ldd].reshape(rows, ldd)
        assert (full[:, V:] == 5.0).all()  # the columns behind the vocabulary stay
        g = full[:, :V]
    return loss[0], row[:rows], g


def check_distill(lib, x, tv, ti, tgt, tau=1.0, alpha=1.0, scale=0.25, **kw):
    V = x.shape[1]
    loss, row, g = run_distill(lib, x, tv, ti, tgt, tau, alpha, scale, **kw)
    rl, rr, rg, size = ref_distill(x, tv, ti, tgt, tau, alpha, scale)
    # Relative error of a probability: the difference to the maximum and its
    # product with 1 / tau are rounded (2 roundings of the exponent, so
    # 2 D roundings of the exponential, and 1 / tau's own: 3 D), the
    # exponentials and logarithms are good to a few steps (8), and a sum of V
    # terms adds one rounding a term in its longest chain (at most V / 128 + 32).
    fin = np.where(np.isfinite(x), x, np.nan)
    with np.errstate(all="ignore"):
        D = np.nanmax(np.nanmax(fin, 1) - np.nanmin(fin, 1)) if np.isfinite(fin).any() else 0.0
    D = max(1.0, float(D) * max(1.0, 1.0 / tau))
    rel = EPS * (3 * D + 8 + V / 128 + 32)
    # row loss: its terms are logarithms of size up to D + log V, each exact to
    # `rel` absolutely and three roundings relatively
    t2 = alpha * tau * tau + (1 - alpha)
    tol_row = t2 * (2 * rel + 6 * EPS * (2 * D + math.log(V) + 16))
    inf = ~np.isfinite(rr)
    assert np.array_equal(np.isinf(row), np.isinf(rr))
    off = np.abs(row[~inf] - rr[~inf]).max(initial=0.0)
    assert off <= tol_row, (off, tol_row)
    if inf.any():
        assert loss == rl
    else:
        n = len(rr)
        assert abs(loss - rl) <= scale * (n * tol_row + (n + 2) * EPS * np.abs(rr).sum())
    if g is not None:
        assert np.isfinite(g).all()
        bad = np.abs(g - rg) > size * (rel + 6 * EPS) + 1e-37
        assert not bad.any(), (np.argwhere(bad)[:4], g[bad][:4], rg[bad][:4])
    return loss, row, g


def teacher(rows, V, k, seed):
    g = np.random.default_rng(seed)
    ti = np.stack([g.permutation(V)[:k] for _ in range(rows)]).astype(np.int32)
    tv = -np.sort(-g.standard_normal((rows, k)) * 3.0, 1)
    return tv.astype(np.float32), ti, g.integers(0, V, rows).astype(np.int32)


@pytest.mark.parametrize("V,k,rows", [(1, 1, 3), (7, 3, 5), (65, 64, 9), (4099, 16, 12), (50257, 64, 6), (50257, 1024, 2),
                                      (50260, 1, 3), (128256, 100, 2), (300001, 33, 2)])
@pytest.mark.parametrize("tau,alpha", [(1.0, 1.0), (2.0, 0.5), (0.5, 0.0), (3.0, 1.0), (1.0, 0.3)])
def test_distill_sizes(lib, cuda, V, k, rows, tau, alpha):
    tv, ti, tgt = teacher(rows, V, k, V + k)
    x = logits(rows, V, k)
    a = check_distill(lib, x, tv, ti, tgt, tau, alpha)
    b = check_distill(lib, x, tv, ti, tgt, tau, alpha, grad=False)
    assert a[0] == b[0] and np.array_equal(a[1], b[1])  # the loss is the same without its gradient
    c = check_distill(lib, x, tv, ti, tgt, tau, alpha, inplace=True)
    assert np.array_equal(a[2], c[2])


@pytest.mark.parametrize("rows,V,k,ld,shift", [(1783, 5, 3, 5, 0), (1783, 513, 40, 515, 1), (1779, 1300, 8, 1300, 0),
                                               (1778, 4096, 64, 4096, 2), (297, 4096, 1024, 4099, 0), (297, 4097, 16, 4097, 3)])
def test_distill_many_short_rows(lib, cuda, rows, V, k, ld, shift):
    tv, ti, tgt = teacher(rows, V, k, V)
    x = logits(rows, V, k)
    x[5], ti[6], tgt[7] = -INF, -1, -1
    ti[8, : k // 2 + 1] = ti[8, 0]  # one token many times
    a = check_distill(lib, x, tv, ti, tgt, 2.0, 0.5, ld=ld, shift=shift)
    b = check_distill(lib, x, tv, ti, tgt, 2.0, 0.5, grad=False, ld=ld, shift=shift)
    assert a[0] == b[0] and np.array_equal(a[1], b[1])
    check_distill(lib, x, tv, ti, tgt, 1.0, 0.7, inplace=True, ld=ld, shift=shift)


@pytest.mark.parametrize("ld,shift,ldd", [(1003, 0, 1003), (1003, 1, 1003), (1004, 2, 1007), (1010, 3, 1003)])
def test_distill_strides_and_alignment(lib, cuda, ld, shift, ldd):
    tv, ti, tgt = teacher(9, 1003, 20, 1)
    x = logits(9, 1003, 2)
    check_distill(lib, x, tv, ti, tgt, 2.0, 0.6, ld=ld, shift=shift, ldd=ldd)
    check_distill(lib, x, tv, ti, tgt, 2.0, 0.6, ld=ld, shift=shift, inplace=True)


@pytest.mark.parametrize("V", [97, 4099, 50257])
@pytest.mark.parametrize("tau,alpha", [(1.0, 0.5), (2.0, 1.0)])
def test_distill_far_below_zero_beside_masked_stretches(lib, cuda, V, tau, alpha):
    """Logits far below 0 next to warps and blocks that hold -inf alone: a part
    without weight must not be scaled by 2^(0 - R)."""
    tv, ti, tgt = teacher(5, V, 8, V)
    x = logits(5, V, V) - np.float32(400.0)
    first = (V + 1) // 2
    x[0, :first], x[1, first:], x[2, : V - 3] = -INF, -INF, -INF
    x[3, np.arange(V) % 1024 < min(128, V // 2)] = -INF  # of some warps every group of four
    for r in range(5):
        live = np.flatnonzero(x[r] > -INF)
        ti[r] = live[np.arange(8) % live.size]
        tgt[r] = live[-1]
    check_distill(lib, x, tv, ti, tgt, tau, alpha)
    check_distill(lib, x, tv, ti, tgt, tau, alpha, grad=False)


@pytest.mark.parametrize("V", [97, 50257])
def test_distill_padding_duplicates_and_empty_rows(lib, cuda, V):
    g = np.random.default_rng(V)
    rows, k = 14, 12
    tv, ti, tgt = teacher(rows, V, k, 3)
    x = logits(rows, V, 4)
    ti[0] = -1                       # no list
    ti[1], tgt[1] = -1, -1           # nothing at all
    tgt[2] = V                       # a target outside the vocabulary
    ti[3, 5:] = V + 7                # list entries outside it
    ti[4] = 5                        # one token all over
    ti[5, ::2] = 9                   # one token several times
    tv[6, 1:] = -INF
    tv[7] = -INF
    tv[8, 3] = NAN
    x[9] = -INF                      # a student row without a finite logit
    x[10, g.random(V) < 0.5] = -INF  # part of the vocabulary masked
    x[10, ti[10]] = 1.0
    x[10, tgt[10]] = 0.5
    tv[11] = 80.0                    # equal and large
    tv[12] = np.linspace(0, -4000, k)
    tgt[13] = ti[13, 0]              # the target is on the list
    for tau, alpha in ((1.0, 1.0), (2.0, 0.5), (1.0, 0.0)):
        check_distill(lib, x, tv, ti, tgt, tau, alpha)
        check_distill(lib, x, tv, ti, tgt, tau, alpha, inplace=True)


def test_distill_masked_teacher_token_makes_the_loss_infinite(lib, cuda):
    tv, ti, tgt = teacher(3, 50, 4, 5)
    x = logits(3, 50, 6)
    x[1, ti[1, 2]] = -INF
    x[2, tgt[2]] = -INF
    ti[2] = -1
    loss, row, g = check_distill(lib, x, tv, ti, tgt, 1.0, 0.5)
    assert np.isinf(row[1]) and np.isinf(row[2]) and np.isfinite(row[0]) and loss == INF


def test_distill_without_lists_is_cross_entropy(lib, cuda):
    """alpha = 0 is the library's own cross-entropy, with its gradient."""
    rows, V = 20, 50257
    x = logits(rows, V, 7)
    tgt = np.random.default_rng(8).integers(0, V, rows).astype(np.int32)
    loss, _, g = check_distill(lib, x, None, None, tgt, 1.0, 0.0, scale=1.0 / rows)
    dx, dt = dev(x), dev(tgt)
    pr, ls = torch.empty(rows, V, device="cuda"), torch.empty(1, device="cuda")
    dl = torch.zeros(rows, V, device="cuda")
    lib.cross_entropy_fwd(ptr(dx), ptr(dt), ptr(pr), ptr(ls), 1, rows, V)
    lib.cross_entropy_bwd(ptr(dl), ptr(pr), ptr(dt), 1.0 / rows, 1, rows, V)
    abi.check(lib, lib.cngpt_cuda_check())
    # both are within the bound of check_distill of the 64-bit value
    assert abs(float(ls[0]) - loss) <= 2e-5 * abs(loss)
    assert np.abs(dl.cpu().numpy() - g).max() <= 1.0 / rows * 1e-4


def test_distill_gradient_against_differences(lib, cuda):
    """Central differences of the 64-bit loss, along random directions."""
    rows, V, k = 4, 211, 9
    tv, ti, tgt = teacher(rows, V, k, 9)
    x = logits(rows, V, 10)
    rng = np.random.default_rng(11)
    for tau, alpha in ((1.0, 1.0), (2.0, 0.4)):
        _, _, g = run_distill(lib, x, tv, ti, tgt, tau, alpha, 1.0)
        for _ in range(5):
            v = rng.standard_normal(x.shape)
            h = 1e-4
            a = ref_distill(x + h * v, tv, ti, tgt, tau, alpha, 1.0)[0]
            b = ref_distill(x - h * v, tv, ti, tgt, tau, alpha, 1.0)[0]
            # the difference's own error: h^2 / 6 times a third derivative of at most
            # (sum |v|)^3-free softmax bounds, about 1e-8 * max |v|^3; the gradient's: 1e-5 of sum |g v|
            assert abs((a - b) / (2 * h) - float((g * v).sum())) <= 1e-5 * float(np.abs(g * v).sum()) + 1e-6


def test_distill_nan_logits_give_nan(lib, cuda):
    tv, ti, tgt = teacher(2, 100, 4, 12)
    x = logits(2, 100, 13)
    x[1, 50] = NAN
    loss, row, g = run_distill(lib, x, tv, ti, tgt, 1.0, 0.5, 1.0)
    assert np.isnan(row[1]) and np.isnan(loss) and np.isfinite(row[0]) and np.isfinite(g[0]).all() and np.isnan(g[1]).any()


def test_distill_without_rows_writes_a_zero_loss(lib, cuda):
    loss = torch.full((1,), 7.0, device="cuda")
    abi.check(lib, lib.cngpt_cuda_distill(None, 10, 0, 10, None, None, 0, None, 1.0, 1.0, 1.0, ptr(loss), None, None, 0))
    abi.check(lib, lib.cngpt_cuda_check())
    assert float(loss[0]) == 0.0


def test_largest_vocabularies(lib, cuda):
    """The most that each entry point takes; one more is refused."""
    x = logits(2, 262144, 30)
    check_sample(lib, x, T=[0.8, 1.1], k=[40, 0], p=[0.9, 0.8], u=[0.3, 0.6])
    x = logits(2, 400000, 31)
    check_topk(lib, x, 70)
    tv, ti, tgt = teacher(2, 400000, 40, 32)
    check_distill(lib, x, tv, ti, tgt, 2.0, 0.5)
    d = dev(x)
    o, i = torch.empty(8, device="cuda"), torch.empty(8, dtype=torch.int32, device="cuda")
    assert lib.cngpt_cuda_topk(ptr(d), 400001, 1, 400001, 2, ptr(o), ptr(i)) == abi.ERR_ARG
    assert lib.cngpt_cuda_distill(ptr(d), 400001, 1, 400001, None, None, 0, ptr(i), 1.0, 0.0, 1.0, ptr(o), ptr(o), None,
                                  0) == abi.ERR_ARG
    assert lib.cngpt_cuda_sample(ptr(d), 262145, 1, 262145, None, None, None, None, ptr(o), ptr(i), None) == abi.ERR_ARG
    lib.cngpt_cuda_clear_status()


def test_distill_overlap_is_refused(lib, cuda):
    d = torch.zeros(4, 64, device="cuda")
    o, i = torch.zeros(8, device="cuda"), torch.zeros(8, dtype=torch.int32, device="cuda")

    def call(out, ldd):
        return lib.cngpt_cuda_distill(ptr(d), 64, 3, 60, None, None, 0, ptr(i), 1.0, 0.0, 1.0, ptr(o), ptr(o), out, ldd)
    assert call(ptr(d) + 4, 64) == abi.ERR_ARG
    assert call(ptr(d), 60) == abi.ERR_ARG
    assert call(ptr(d) + 4 * 64, 64) == abi.ERR_ARG
    assert call(ptr(torch.zeros(4, 64, device="cuda")), 59) == abi.ERR_ARG
    assert call(ptr(d), 64) == abi.OK
    lib.cngpt_cuda_clear_status()


# ---------------------------------------------------------- streams, graphs
def test_operators_on_another_stream_and_in_a_graph(lib, cuda):
    """Captured once, replayed on new inputs in the same buffers: the results
    of eager calls, on a stream of the caller's own."""
    rows, V, k = 6, 50257, 16
    x = torch.empty(rows, V, device="cuda")
    u = torch.empty(rows, device="cuda")
    T, tk, tp = torch.full((rows,), 0.8, device="cuda"), torch.full((rows,), 50, dtype=torch.int32, device="cuda"), \
        torch.full((rows,), 0.9, device="cuda")
    tgt = torch.zeros(rows, dtype=torch.int32, device="cuda")

    def bufs():
        return dict(tok=torch.empty(rows, dtype=torch.int32, device="cuda"), lp=torch.empty(rows, device="cuda"),
                    v=torch.empty(rows, k, device="cuda"), i=torch.empty(rows, k, dtype=torch.int32, device="cuda"),
                    loss=torch.empty(1, device="cuda"), row=torch.empty(rows, device="cuda"),
                    d=torch.empty(rows, V, device="cuda"))

    def calls(o):
        abi.check(lib, lib.cngpt_cuda_sample(ptr(x), V, rows, V, ptr(T), ptr(tk), ptr(tp), None, ptr(u), ptr(o["tok"]),
                                             ptr(o["lp"])))
        abi.check(lib, lib.cngpt_cuda_topk(ptr(x), V, rows, V, k, ptr(o["v"]), ptr(o["i"])))
        abi.check(lib, lib.cngpt_cuda_distill(ptr(x), V, rows, V, ptr(o["v"]), ptr(o["i"]), k, ptr(tgt), 2.0, 0.5, 1.0,
                                              ptr(o["loss"]), ptr(o["row"]), ptr(o["d"]), V))

    a, b = bufs(), bufs()
    g = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    x.normal_()
    u.uniform_()
    torch.cuda.synchronize()
    try:
        with torch.cuda.graph(g, stream=side):
            lib.cngpt_cuda_set_stream(side.cuda_stream)
            calls(a)
        for seed in range(3):
            torch.manual_seed(seed)
            x.normal_()
            u.uniform_()
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                g.replay()
                calls(b)
            side.synchronize()
            for n in a:
                assert torch.equal(a[n], b[n]), n
    finally:
        lib.cngpt_cuda_set_stream(None)


def test_offsets_beyond_32_bits(lib, cuda):
    """Rows that start more than 2^31 floats into the buffer."""
    V, ld = 50257, 1 << 30
    buf = torch.empty(2 * ld + V, device="cuda")
    x = logits(3, V, 20)
    for r in range(3):
        buf[r * ld:r * ld + V] = torch.from_numpy(x[r]).cuda()
    u = np.array([0.2, 0.7, 0.9], np.float32)
    du, tok = dev(u), torch.empty(3, dtype=torch.int32, device="cuda")
    v, i = torch.empty(3, 5, device="cuda"), torch.empty(3, 5, dtype=torch.int32, device="cuda")
    loss, row = torch.empty(1, device="cuda"), torch.empty(3, device="cuda")
    abi.check(lib, lib.cngpt_cuda_sample(ptr(buf), ld, 3, V, None, None, None, None, ptr(du), ptr(tok), None))
    abi.check(lib, lib.cngpt_cuda_topk(ptr(buf), ld, 3, V, 5, ptr(v), ptr(i)))
    abi.check(lib, lib.cngpt_cuda_distill(ptr(buf), ld, 3, V, ptr(v), ptr(i), 5, None, 1.0, 1.0, 1.0, ptr(loss), ptr(row),
                                          ptr(buf), ld))
    abi.check(lib, lib.cngpt_cuda_check())
    assert tok.cpu().tolist() == [ref_sample(x[r], 1.0, 0, 1.0, 0.0, float(u[r]))[0] for r in range(3)]
    rv, ri = ref_topk(x, 5)
    assert np.array_equal(i.cpu().numpy(), ri)
    _, _, rg, size = ref_distill(x, rv, ri, None, 1.0, 1.0, 1.0)
    for r in range(3):
        got = buf[r * ld:r * ld + V].cpu().numpy()
        assert (np.abs(got - rg[r]) <= size[r] * EPS * (3 * 25 + 8 + V / 128 + 38) + 1e-37).all()
