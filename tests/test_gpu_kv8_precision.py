"""Precision of attention over the 8-bit cache in every row type: operands and
weights as good as f32's, one rounding at the end.

Bounds (u = 2^-24): a score is off by (head_dim + 32) u S, S the largest
scale x sum |q_i k_i|, a weight by twice that relatively and by 2^-22 as a
pair of f16, so the weighted sum by 2 x the scores' part + 64 u of V = max |v|;
the tensor cores' running sum is cut, not rounded, at each of n / 16 steps of
two products (2 u each, of V). Then half a step of the type."""
import numpy as np
import pytest

import hotseat_b200 as hs
from kv8_ref import Cache
from test_gpu_kv8 import DT, U, dev, i32

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def bound(want, size, top, hd, n, dtype):
    e = 4 * (hd + 32) * U * size * top + 64 * U * top + n / 8 * 2 * U * top
    return e + (np.abs(want) + e) * torch.finfo(DT[dtype]).eps / 2 + torch.finfo(DT[dtype]).tiny


def close(got, want, size, top, hd, n, dtype):
    err = np.abs(got.astype(np.float64) - want)
    worst = np.max(err / bound(want, size, top, hd, n, dtype))
    assert worst <= 1, worst


def run(form, s, q, n):
    """Rows of q as the last ones of n cached positions of one slot: each by itself, or as one chunk."""
    out = torch.full_like(q, 9.0)
    m = q.shape[0]
    if form == "chunk":
        s.attend(0, q, out, i32([n - m]), i32([0, m]))
    else:
        for r in range(m):
            s.attend(0, q[r:r + 1], out[r:r + 1], i32([n - m + r]))
    s.check()
    return out.float().cpu().numpy()


FORMS = ["single", "chunk"]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd, nh, nkv", [(64, 7, 1), (128, 12, 2)])
def test_weights_that_cancel(form, dtype, hd, nh, nkv):
    """V of +1 and -1 in turn: the result is a small difference of sums, and keeps what the weights hold."""
    rng = np.random.default_rng(hd)
    n = 40
    kv, ref = hs.Kv.alloc8(hs.KvSpec(1, nkv, hd, n, 0)), Cache(nkv, hd, n, 1)
    s = hs.Kv8Set([kv], n_heads=nh)
    k = rng.standard_normal((n, nkv, hd)).astype(np.float32)
    v = (np.where(np.arange(n) % 2, -1.0, 1.0)[:, None, None] * np.ones((n, nkv, hd))).astype(np.float32)
    s.append(0, dev(k), dev(v), i32([0]), i32([0, n]))
    ref.append(0, k, v)
    q = dev((rng.standard_normal((n, nh, hd)) * 0.2).astype(np.float32), DT[dtype])
    got, qf = run(form, s, q, n), q.float().cpu().numpy()
    for r in range(n):
        close(got[r], *ref.attend(qf[r], r, hd ** -0.5), hd, r + 1, dtype)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd, nh, nkv, block", [(64, 7, 1, 1), (128, 12, 2, 16)])
def test_large_scores_near_one_another(form, dtype, hd, nh, nkv, block):
    """Scores of about 16 whose differences decide: a score that is off by a part of itself shows."""
    rng = np.random.default_rng(hd + 1)
    n = 48
    kv, ref = hs.Kv.alloc8(hs.KvSpec(1, nkv, hd, n, 0), block=block), Cache(nkv, hd, n, block)
    s = hs.Kv8Set([kv], n_heads=nh)
    way = np.where(rng.random((1, nkv, hd)) < 0.5, -1.0, 1.0)
    k = (way * (1 + 0.02 * rng.standard_normal((n, nkv, 1)))).astype(np.float32)
    v = (np.where(np.arange(n) % 2, -1.0, 1.0)[:, None, None] * (1 + 0.2 * rng.random((n, nkv, hd)))).astype(np.float32)
    s.append(0, dev(k), dev(v), i32([0]), i32([0, n]))
    ref.append(0, k, v)
    q = np.repeat(way, nh // nkv, axis=1) * (16 * hd ** -0.5) * (1 + 0.01 * rng.standard_normal((n, nh, 1)))
    q = dev(q.astype(np.float32), DT[dtype])
    got, qf = run(form, s, q, n), q.float().cpu().numpy()
    for r in range(n):
        close(got[r], *ref.attend(qf[r], r, hd ** -0.5), hd, r + 1, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("times", [2.0 ** 12, 2.0 ** 40, 2.0 ** 90])
@pytest.mark.parametrize("hd, nh, nkv, block, n, lo, rise", [
    (64, 7, 1, 1, 300, 100, 200), (128, 12, 2, 16, 300, 100, 160), (64, 4, 2, 1, 290, 0, 1), (64, 3, 1, 1, 4400, 4110, 4300),
    (128, 2, 2, 32, 4300, 4100, 4128)])
def test_large_values_behind_a_row_do_not_reach_it(dtype, times, hd, nh, nkv, block, n, lo, rise):
    """K and V from position `rise` on are far larger than before it: rows before it keep their precision."""
    rng = np.random.default_rng(n + hd)
    kv, ref = hs.Kv.alloc8(hs.KvSpec(1, nkv, hd, n, 0), block=block), Cache(nkv, hd, n, block)
    s = hs.Kv8Set([kv], n_heads=nh)
    k, v = (rng.standard_normal((n, nkv, hd)).astype(np.float32) for _ in range(2))
    k[rise:] *= np.float32(times)
    v[rise:] *= np.float32(times)
    s.append(0, dev(k), dev(v), i32([0]), i32([0, n]))
    ref.append(0, k, v)
    q = dev((rng.standard_normal((n - lo, nh, hd)) * 0.3).astype(np.float32), DT[dtype])
    out = torch.empty_like(q)
    s.attend(0, q, out, i32([lo]), i32([0, n - lo]))
    s.check()
    got, qf = out.float().cpu().numpy(), q.float().cpu().numpy()
    for p in sorted({lo, rise - 1, (lo + rise) // 2, max(lo, rise - 7)}):
        close(got[p - lo], *ref.attend(qf[p - lo], p, hd ** -0.5), hd, p + 1, dtype)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("size", [2.0 ** 22, 2.0 ** 26, 2.0 ** 45, 2.0 ** 100])
@pytest.mark.parametrize("hd, nh, nkv", [(64, 7, 1), (128, 4, 2)])
def test_scores_of_any_size(form, dtype, size, hd, nh, nkv):
    """Scores of about `size`, the largest by a third: it takes all the weight. And rows whose scores are all alike."""
    rng = np.random.default_rng(hd + 2)
    n, m = 200, 60
    kv, ref = hs.Kv.alloc8(hs.KvSpec(1, nkv, hd, n, 0)), Cache(nkv, hd, n, 1)
    s = hs.Kv8Set([kv], n_heads=nh)
    way = np.where(rng.random((1, nkv, hd)) < 0.5, -1.0, 1.0)
    k = way * rng.uniform(0.25, 0.6, (n, nkv, 1))
    k[100] = way[0]
    v = rng.standard_normal((n, nkv, hd)).astype(np.float32)
    k = k.astype(np.float32)
    s.append(0, dev(k), dev(v), i32([0]), i32([0, n]))
    ref.append(0, k, v)
    # odd factors, so that no product of them is exact
    q = np.repeat(way, nh // nkv, axis=1) * rng.uniform(1.1, 1.9, (m, nh, 1))
    q = dev(q.astype(np.float32), DT[dtype])
    scale = float(np.float32(size * 1.2345 / hd))
    out = torch.full_like(q, 9.0)
    one = lambda o: s.attend(0, q, o, i32([n - m]), i32([0, m]), scale=scale)  # noqa: E731
    if form == "single":
        one = lambda o: [s.attend(0, q[r:r + 1], o[r:r + 1], i32([n - m + r]), scale=scale) for r in range(m)]  # noqa: E731
    one(out)
    got = out.float().cpu().numpy()
    top = ref.values(1, 100, 101)[0].astype(np.float64)[np.arange(nh) // (nh // nkv)]
    err = np.abs(got - top) - np.abs(top) * torch.finfo(DT[dtype]).eps / 2
    assert np.all(err <= 64 * U * np.abs(top).max()), np.max(err)
    k[:] = k[:1]
    s.append(0, dev(k), dev(v), i32([0]), i32([0, n]))
    one(out)
    got = out.float().cpu().numpy()
    vals = ref.values(1, 0, n).astype(np.float64)
    for r in (0, m - 1):
        want = vals[:n - m + r + 1].mean(0)[np.arange(nh) // (nh // nkv)]
        assert np.all(np.abs(got[r] - want) <= bound(want, 0, np.abs(vals).max(), hd, n, dtype))
