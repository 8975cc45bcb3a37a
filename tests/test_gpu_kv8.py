"""The 8-bit KV cache on the GPU: rows quantised and read back bit for bit as
restated (kv8_ref), and attention over it against 64 bits.

Error bounds of attention, from arithmetic alone (u = 2^-24): a score is a
sum of head_dim products of f32 precision, off by at most (head_dim + 32) u S,
S the largest scale x sum |q_i k_i|; weights then by 2 x that relatively
(numerator and sum), the weighted sum of values by as much of V = max |v|,
and its own summation and the splits' joins by 64 u V. 16-bit inputs may round each
weight once to f16 (2^-11 V) and round the result once (half a step)."""
import numpy as np
import pytest

import hotseat_b200 as hs
from kv8_ref import Cache

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def rows_of(rng, m, heads, hd, dtype, spread=1.0):
    """Rows in `dtype` on the GPU and their exact f32 values here."""
    x = rng.standard_normal((m, heads, hd)) * np.exp(rng.uniform(-spread, spread, (m, heads, 1)))
    t = dev(x.astype(np.float32), DT[dtype])
    return t, t.float().cpu().numpy()


def raw(kv, layer=0):
    """(codes [2][max_ctx][nkv][hd], scales [2][blocks][nkv]) of a region's layer, by its layout."""
    s, block = kv.spec, kv.block
    nb = -(-s.max_ctx // block)
    pad = lambda n: -(-n // 256) * 256  # noqa: E731
    plane, splane = pad(s.max_ctx * s.n_kv_heads * s.head_dim), pad(nb * s.n_kv_heads * 4)
    at = layer * 2 * (plane + splane)
    codes, scales = [], []
    for w in range(2):
        c = kv.read(at + w * plane, s.max_ctx * s.n_kv_heads * s.head_dim).view(np.int8)
        f = kv.read(at + 2 * plane + w * splane, nb * s.n_kv_heads * 4).view(np.float32)
        if s.layout == hs.TOKEN_MAJOR:
            codes.append(c.reshape(s.max_ctx, s.n_kv_heads, s.head_dim))
            scales.append(f.reshape(nb, s.n_kv_heads))
        else:
            codes.append(c.reshape(s.n_kv_heads, s.max_ctx, s.head_dim).transpose(1, 0, 2))
            scales.append(f.reshape(s.n_kv_heads, nb).T)
    return np.stack(codes), np.stack(scales)


def same(kv, ref, layer=0):
    codes, scales = raw(kv, layer)
    assert np.array_equal(scales.view(np.uint32) & 0x7FFFFFFF if np.isnan(ref.scales).any() else scales,
                          ref.scales.view(np.uint32) & 0x7FFFFFFF if np.isnan(ref.scales).any() else ref.scales)
    assert np.array_equal(codes, ref.codes)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("block, layout, hd", [(1, 0, 64), (1, 1, 128), (16, 0, 128), (32, 1, 64), (64, 0, 64),
                                               (64, 1, 128), (128, 0, 64), (128, 1, 128)])
def test_append_and_read_are_exact(dtype, block, layout, hd):
    """Ragged chunks, single rows, an empty slot, a second layer, rows past the last sequence."""
    rng = np.random.default_rng(block * 7 + hd)
    nkv, max_ctx = 3, 301
    spec = hs.KvSpec(2, nkv, hd, max_ctx, layout)
    kvs = [hs.Kv.alloc8(spec, block=block) for _ in range(4)]
    refs = [[Cache(nkv, hd, max_ctx, block) for _ in kvs] for _ in range(2)]
    s = hs.Kv8Set(kvs)
    at = [0, 0, 0, 0]
    for counts in ([70, 1, 0, 129], [5, 33, 16, 0], [1, 1, 1, 1], [100, 2, 200, 31]):
        for layer in (0, 1):
            m = sum(counts)
            k, kf = rows_of(rng, m + 2, nkv, hd, dtype)
            v, vf = rows_of(rng, m + 2, nkv, hd, dtype)
            start = np.concatenate([[0], np.cumsum(counts)])
            s.append(layer, k, v, i32(at), i32(start))
            for i in range(4):
                refs[layer][i].append(at[i], kf[start[i]:start[i + 1]], vf[start[i]:start[i + 1]])
        at = [a + c for a, c in zip(at, counts)]
    s.check()
    for layer in (0, 1):
        for kv, ref in zip(kvs, refs[layer]):
            same(kv, ref, layer)
    # read back from odd places, into rows that others lie behind
    lo, n = [3, 0, 150, 17], [64, 30, 1, 0]
    start = np.concatenate([[0], np.cumsum(n)])
    k = torch.full((sum(n) + 3, nkv, hd), 7.0, dtype=DT[dtype], device="cuda")
    v = torch.full_like(k, 7.0)
    s.read(1, k, v, i32(lo), i32(start))
    for which, t in ((0, k), (1, v)):
        for i in range(4):
            want = torch.from_numpy(refs[1][i].values(which, lo[i], lo[i] + n[i])).to(DT[dtype])
            assert torch.equal(t[start[i]:start[i + 1]].cpu(), want)
        assert bool((t[sum(n):] == 7.0).all())


@pytest.mark.parametrize("block", [1, 32])
def test_single_rows_fill_a_cache(block):
    """Decode steps: a row per slot and call, scales growing inside the blocks."""
    rng = np.random.default_rng(3)
    spec = hs.KvSpec(1, 2, 64, 80, 0)
    kvs = [hs.Kv.alloc8(spec, block=block) for _ in range(3)]
    refs = [Cache(2, 64, 80, block) for _ in kvs]
    s = hs.Kv8Set(kvs)
    at = [0, 11, 40]
    for step in range(40):
        k, kf = rows_of(rng, 3, 2, 64, "f32", spread=3.0)
        v, vf = rows_of(rng, 3, 2, 64, "f32", spread=3.0)
        pos = [a + step for a in at]
        if step % 7 == 3:
            pos[1] = -1  # a slot that sits this step out
        s.append(0, k, v, i32(pos))
        for i, p in enumerate(pos):
            if p >= 0:
                refs[i].append(p, kf[i:i + 1], vf[i:i + 1])
    s.check()
    for kv, ref in zip(kvs, refs):
        same(kv, ref)


@pytest.mark.parametrize("block", [1, 16])
def test_values_on_the_border_between_codes(block):
    """Every half step and its neighbours in f32, for scales that divide badly."""
    spec = hs.KvSpec(1, 1, 64, 512, 0)
    kv, ref = hs.Kv.alloc8(spec, block=block), Cache(1, 64, 512, block)
    s = hs.Kv8Set([kv])
    rng = np.random.default_rng(5)
    rows = np.zeros((512, 1, 64), np.float32)
    for r in range(0, 512, block):
        top = np.float32(rng.uniform(0.1, 300) if r else 127.0)
        step = np.float32(top / np.float32(127.0))
        c = rng.integers(-127, 126, size=(block, 63))
        half = ((c + 0.5) * np.float64(step)).astype(np.float32)
        half = np.where(rng.random(half.shape) < 0.33, np.nextafter(half, np.float32(np.inf)), half)
        half = np.where(rng.random(half.shape) < 0.33, np.nextafter(half, np.float32(-np.inf)), half)
        rows[r:r + block, 0, :63] = half
        rows[r:r + block, 0, 63] = top
    s.append(0, dev(rows), dev(-rows), i32([0]), i32([0, 512]))
    ref.append(0, rows, -rows)
    same(kv, ref)


def test_extreme_and_non_finite_rows():
    spec = hs.KvSpec(1, 1, 64, 64, 0)
    for block in (1, 16):
        kv, ref = hs.Kv.alloc8(spec, block=block), Cache(1, 64, 64, block)
        s = hs.Kv8Set([kv])
        rows = np.ones((64, 1, 64), np.float32)
        rows[1] = 0
        rows[2] = 3.4e38
        rows[3] = 1e-45
        rows[4] = 2e-36
        rows[5, 0, 7] = np.inf
        rows[16 + 3, 0, 0] = -np.inf
        rows[32 + 1, 0, 63] = np.nan
        rows[48:] = 0
        for p in range(0, 64):
            s.append(0, dev(rows[p:p + 1]), dev(rows[p:p + 1]), i32([p]))
            ref.append(p, rows[p:p + 1], rows[p:p + 1])
        same(kv, ref)
        k = torch.empty(64, 1, 64, device="cuda")
        s.read(0, k, None, i32([0]), i32([0, 64]))
        assert torch.equal(torch.isnan(k).cpu(), torch.from_numpy(np.isnan(ref.values(0, 0, 64))))


def test_rows_past_max_ctx_are_flagged_and_skipped():
    spec = hs.KvSpec(1, 2, 64, 40, 0)
    for block in (1, 16):
        kv, ref = hs.Kv.alloc8(spec, block=block), Cache(2, 64, 40, block)
        s = hs.Kv8Set([kv], n_heads=2)
        rng = np.random.default_rng(1)
        k, kf = rows_of(rng, 60, 2, 64, "f32")
        s.append(0, k, k, i32([0]), i32([0, 60]))
        ref.append(0, kf, kf)
        with pytest.raises(hs.HotseatError) as e:
            s.check()
        assert e.value.code == hs.HS_E_ARG
        s.check()  # cleared
        same(kv, ref)
        got = torch.full((60, 2, 64), 5.0, device="cuda")
        s.read(0, got, None, i32([0]), i32([0, 60]))
        assert bool((got[40:] == 5.0).all()) and torch.equal(got[:40].cpu(), torch.from_numpy(ref.values(0, 0, 40)))
        with pytest.raises(hs.HotseatError):
            s.check()
        out = torch.full((60, 2, 64), 5.0, device="cuda")
        s.attend(0, k, out, i32([0]), i32([0, 60]))
        assert bool((out[40:] == 0).all()) and not bool((out[:40] == 5.0).any())
        with pytest.raises(hs.HotseatError):
            s.check()
        for pos in (40, 2 ** 31 - 1, -2):  # -2: 2^32 - 2
            s.append(0, k[:1], k[:1], i32([pos]))
            with pytest.raises(hs.HotseatError):
                s.check()
        same(kv, ref)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strided_and_unaligned_rows(dtype):
    """q, k, v as slices of one fused row, heads behind one another or rows, and bases off 16 bytes."""
    rng = np.random.default_rng(9)
    spec = hs.KvSpec(1, 2, 64, 32, 1)
    m, width = 20, 4 * 64 + 2 * 64 + 2 * 64
    for off in (0, 1, 8):
        fused = dev(rng.standard_normal(m * (width + off) + off).astype(np.float32), DT[dtype])
        fused = fused[off:].view(m, width + off)
        k = fused[:, 256:384].unflatten(1, (2, 64))
        v = fused[:, 384:512].unflatten(1, (2, 64))
        kv, ref = hs.Kv.alloc8(spec, block=16), Cache(2, 64, 32, 16)
        s = hs.Kv8Set([kv])
        s.append(0, k, v, i32([0]), i32([0, m]))
        ref.append(0, k.float().cpu().numpy(), v.float().cpu().numpy())
        same(kv, ref)
        back = torch.zeros(2, m + off, 64, dtype=DT[dtype], device="cuda").transpose(0, 1)[:m]
        flat = torch.zeros(2 * m * 64 + off, dtype=DT[dtype], device="cuda")
        s.read(0, back, None, i32([0]), i32([0, m]))
        s.read(0, None, flat[off:].view(m, 2, 64), i32([0]), i32([0, m]))
        assert torch.equal(back.cpu(), torch.from_numpy(ref.values(0, 0, m)).to(DT[dtype]))
        assert torch.equal(flat[off:].view(m, 2, 64).cpu(), torch.from_numpy(ref.values(1, 0, m)).to(DT[dtype]))


def test_dirty_pages_cover_what_changed():
    rng = np.random.default_rng(2)
    for block, layout in ((1, 0), (16, 1), (64, 0)):
        spec = hs.KvSpec(2, 2, 64, 200, layout)
        kv = hs.Kv.alloc8(spec, block=block, page_size=256)
        s = hs.Kv8Set([kv])
        k, _ = rows_of(rng, 70, 2, 64, "f32")
        s.append(1, k, k, i32([0]), i32([0, 70]))
        torch.cuda.synchronize()
        before = kv.read(0, kv.bytes)
        kv.arm()
        big = k[:3] * 100.0
        s.append(1, big, big, i32([70]), i32([0, 3]))
        torch.cuda.synchronize()
        after = kv.read(0, kv.bytes)
        words = kv.harvest()
        marked = np.unpackbits(words.view(np.uint8), bitorder="little")[: kv.n_pages].astype(bool)
        pages = np.nonzero(before != after)[0] // 256
        assert marked[pages].all()
        live = hs.live_ranges_between8(spec, block, 70, 73)
        inside = np.zeros(kv.bytes, bool)
        for off, n in live:
            inside[off:off + n] = True
        assert inside[before != after].all()  # what a hand-over of the new positions would send
        assert 0 < marked.sum() <= 2 * (3 * 2 + 2 + (block + 3) * 2)
        kv.disarm()


# ------------------------------------------------------------------ attention

def filled(rng, lens, nkv, hd, block, layout, max_ctx=None, layers=1, layer=0):
    spec = hs.KvSpec(layers, nkv, hd, max_ctx or max(lens), layout)
    kvs = [hs.Kv.alloc8(spec, block=block) for _ in lens]
    refs = [Cache(nkv, hd, spec.max_ctx, block) for _ in lens]
    s = hs.Kv8Set(kvs)
    k, kf = rows_of(rng, sum(lens), nkv, hd, "f32", spread=0.5)
    v, vf = rows_of(rng, sum(lens), nkv, hd, "f32", spread=1.0)
    start = np.concatenate([[0], np.cumsum(lens)])
    s.append(layer, k, v, i32([0] * len(lens)), i32(start))
    for i, r in enumerate(refs):
        r.append(0, kf[start[i]:start[i + 1]], vf[start[i]:start[i + 1]])
    return kvs, refs


def bound(want, size, top, hd, dtype):
    tol = 2 * (hd + 32) * U * size * 2 * top + 64 * U * top
    if dtype != "f32":
        tol = tol + 2.0 ** -11 * top + np.abs(want) * torch.finfo(DT[dtype]).eps / 2 + torch.finfo(DT[dtype]).tiny
    return tol


def check_rows(got, q, refs, places, scale, dtype):
    """got, q [rows, nh, hd] (numpy, exact values); places: (slot, pos) of each row."""
    for r, (slot, pos) in enumerate(places):
        want, size, top = refs[slot].attend(q[r], pos, scale)
        err = np.abs(got[r].astype(np.float64) - want)
        assert np.all(err <= bound(want, size, top, q.shape[2], dtype)), (r, slot, pos, err.max())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nh, nkv, hd, block, layout", [(14, 2, 64, 1, 0), (12, 2, 128, 32, 1), (3, 3, 64, 16, 1),
                                                        (8, 1, 128, 64, 0), (20, 2, 64, 128, 0), (33, 1, 128, 1, 0)])
def test_single_rows_attend(dtype, nh, nkv, hd, block, layout):
    rng = np.random.default_rng(nh * 100 + hd)
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 257, 700, 1025]
    kvs, refs = filled(rng, lens, nkv, hd, block, layout)
    s = hs.Kv8Set(kvs, n_heads=nh)
    q, qf = rows_of(rng, len(lens), nh, hd, dtype)
    out = torch.empty_like(q)
    s.attend(0, q, out, i32([n - 1 for n in lens]))
    s.check()
    check_rows(out.float().cpu().numpy(), qf, refs, [(i, n - 1) for i, n in enumerate(lens)], hd ** -0.5, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nh, nkv, hd, block, layout", [(14, 2, 64, 1, 0), (12, 2, 128, 32, 1), (2, 2, 128, 16, 0),
                                                        (9, 1, 64, 64, 1), (40, 1, 64, 1, 0)])
def test_ragged_chunks_attend(dtype, nh, nkv, hd, block, layout):
    """Prompts and chunks behind cached positions, single rows, an empty slot, rows behind the last sequence."""
    rng = np.random.default_rng(nh + hd)
    lens = [130, 1, 300, 64, 517, 40]
    rows = [130, 1, 7, 0, 150, 33]
    kvs, refs = filled(rng, lens, nkv, hd, block, layout)
    s = hs.Kv8Set(kvs, n_heads=nh)
    start = np.concatenate([[0], np.cumsum(rows)])
    q, qf = rows_of(rng, sum(rows) + 5, nh, hd, dtype)
    out = torch.full_like(q, 9.0)
    s.attend(0, q, out, i32([n - m for n, m in zip(lens, rows)]), i32(start))
    s.check()
    assert bool((out[sum(rows):] == 9.0).all())
    places = [(i, n - m + j) for i, (n, m) in enumerate(zip(lens, rows)) for j in range(m)]
    pick = sorted(set(list(range(0, len(places), 13)) + [0, 129, 130, 131, 137, 138, 287, 288, len(places) - 1]))
    check_rows(out.float().cpu().numpy()[pick], qf[pick], refs, [places[i] for i in pick], hd ** -0.5, dtype)


def test_a_slot_without_a_position_gives_zeros():
    rng = np.random.default_rng(4)
    kvs, refs = filled(rng, [70, 70, 70], 2, 64, 1, 0)
    s = hs.Kv8Set(kvs, n_heads=4)
    q, qf = rows_of(rng, 3, 4, 64, "f32")
    out = torch.full_like(q, 9.0)
    s.attend(0, q, out, i32([69, -1, 5]))
    assert bool((out[1] == 0).all())
    check_rows(out.cpu().numpy()[[0, 2]], qf[[0, 2]], refs, [(0, 69), (2, 5)], 0.125, "f32")
    q, qf = rows_of(rng, 30, 4, 64, "f32")
    out = torch.full_like(q, 9.0)
    s.attend(0, q, out, i32([60, -1, 5]), i32([0, 10, 20, 30]))
    assert bool((out[10:20] == 0).all())
    check_rows(out.cpu().numpy()[[0, 9, 29]], qf[[0, 9, 29]], refs, [(0, 60), (0, 69), (2, 14)], 0.125, "f32")
    s.check()


@pytest.mark.parametrize("form", ["single", "chunk"])
def test_rows_behind_the_position_are_not_seen(form):
    """Positions behind a row's own hold NaN scales; the results do not change."""
    rng = np.random.default_rng(6)
    for hd, block in ((64, 1), (128, 16)):
        kvs, refs = filled(rng, [400], 2, hd, block, 0)
        s = hs.Kv8Set(kvs, n_heads=6)
        pos = 64 + block - 1 if form == "single" else 64
        m = 1 if form == "single" else 96 - 64
        q, _ = rows_of(rng, m, 6, hd, "f32")
        out, again = torch.empty_like(q), torch.empty_like(q)
        start = None if form == "single" else i32([0, m])
        s.attend(0, q, out, i32([pos]), start)
        bad = torch.full((400 - 96, 2, hd), float("nan"), device="cuda")
        s.append(0, bad, bad, i32([96]), i32([0, 400 - 96]))
        s.attend(0, q, again, i32([pos]), start)
        assert torch.equal(out, again) and bool(torch.isfinite(out).all())


def test_a_stored_infinity_reaches_only_the_rows_that_see_it():
    rng = np.random.default_rng(8)
    kvs, refs = filled(rng, [200], 1, 64, 1, 0)
    s = hs.Kv8Set(kvs, n_heads=2)
    bad = torch.ones(1, 1, 64, device="cuda")
    bad[0, 0, 3] = float("inf")
    good = torch.ones(1, 1, 64, device="cuda")
    s.append(0, good, bad, i32([100]))
    q, _ = rows_of(rng, 200, 2, 64, "f32")
    out = torch.empty_like(q)
    s.attend(0, q, out, i32([0]), i32([0, 200]))
    assert bool(torch.isfinite(out[:100]).all()) and bool(torch.isnan(out[100:]).all())
    one = torch.empty_like(q[:1])
    for p, seen in ((99, False), (100, True), (199, True)):
        s.attend(0, q[:1], one, i32([p]))
        assert bool(torch.isnan(one).all()) == seen


@pytest.mark.parametrize("size", [1e-30, 1e-6, 1.0, 1e4, 1e30])
def test_scales_and_queries_of_any_size(size):
    """Large and tiny K, V and q, with the softmax scale to match."""
    rng = np.random.default_rng(10)
    spec = hs.KvSpec(1, 1, 64, 150, 0)
    for qs in (1.0, 1e-20, 1e20):
        kv, ref = hs.Kv.alloc8(spec), Cache(1, 64, 150, 1)
        s = hs.Kv8Set([kv], n_heads=3)
        k = (rng.standard_normal((150, 1, 64)) * size).astype(np.float32)
        v = (rng.standard_normal((150, 1, 64)) * size).astype(np.float32)
        v[::7] *= np.float32(1e-4)
        s.append(0, dev(k), dev(v), i32([0]), i32([0, 150]))
        ref.append(0, k, v)
        q = (rng.standard_normal((150, 3, 64)) * qs).astype(np.float32)
        scale = 0.125 / (size * qs)
        if not 1e-37 < scale < 1e38:
            continue
        scale = float(np.float32(scale))
        out = torch.empty(150, 3, 64, device="cuda")
        s.attend(0, dev(q), out, i32([0]), i32([0, 150]), scale=scale)
        check_rows(out.cpu().numpy()[[0, 1, 149]], q[[0, 1, 149]], [ref], [(0, 0), (0, 1), (0, 149)], scale, "f32")
        s.attend(0, dev(q[149:]), out[:1], i32([149]), scale=scale)
        check_rows(out.cpu().numpy()[:1], q[149:], [ref], [(0, 149)], scale, "f32")


def test_peaked_scores():
    """One position takes all the weight, and scores far below the largest."""
    rng = np.random.default_rng(12)
    kvs, refs = filled(rng, [900], 2, 64, 1, 0)
    s = hs.Kv8Set(kvs, n_heads=4)
    q, qf = rows_of(rng, 900, 4, 64, "f32")
    out = torch.empty_like(q)
    s.attend(0, q, out, i32([0]), i32([0, 900]), scale=40.0)
    pick = [0, 5, 500, 899]
    check_rows(out.cpu().numpy()[pick], qf[pick], refs, [(0, p) for p in pick], 40.0, "f32")
    s.attend(0, q[899:], out[:1], i32([899]), scale=40.0)
    check_rows(out.cpu().numpy()[:1], qf[899:], refs, [(0, 899)], 40.0, "f32")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd, nh, nkv, n", [(64, 14, 2, 32768), (128, 12, 2, 32768), (128, 4, 1, 70001)])
def test_long_contexts(dtype, hd, nh, nkv, n):
    rng = np.random.default_rng(n)
    kvs, refs = filled(rng, [n], nkv, hd, 16, 0)
    s = hs.Kv8Set(kvs, n_heads=nh)
    q, qf = rows_of(rng, 9, nh, hd, dtype)
    out = torch.empty_like(q)
    s.attend(0, q, out, i32([n - 9]), i32([0, 9]))
    check_rows(out.float().cpu().numpy()[[0, 8]], qf[[0, 8]], refs, [(0, n - 9), (0, n - 1)], hd ** -0.5, dtype)
    s.attend(0, q[8:], out[:1], i32([n - 1]))
    check_rows(out.float().cpu().numpy()[:1], qf[8:], refs, [(0, n - 1)], hd ** -0.5, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nh, nkv, hd, block, layout", [(14, 2, 64, 1, 0), (12, 2, 128, 32, 1), (5, 1, 128, 1, 0)])
def test_few_rows_behind_long_contexts(dtype, nh, nkv, hd, block, layout):
    """Chunks whose positions a cluster shares: slots at and around where it begins, with short and long chunks beside
    them, one that runs past max_ctx, and each alone with the same bits."""
    rng = np.random.default_rng(nh * hd)
    lens, rows = [4099, 4135, 9001, 300, 4097, 9000], [3, 40, 130, 60, 1, 20]
    kvs, refs = filled(rng, lens, nkv, hd, block, layout)
    s = hs.Kv8Set(kvs, n_heads=nh)
    start = np.concatenate([[0], np.cumsum(rows)])
    pos = [n - m for n, m in zip(lens, rows)]
    pos[5] += 4  # its last three rows lie past max_ctx (9,001)
    q, qf = rows_of(rng, sum(rows) + 3, nh, hd, dtype)
    out = torch.full_like(q, 9.0)
    s.attend(0, q, out, i32(pos), i32(start))
    with pytest.raises(hs.HotseatError):
        s.check()
    assert bool((out[sum(rows):] == 9.0).all()) and bool((out[sum(rows) - 3:sum(rows)] == 0).all())
    places = [(i, pos[i] + j) for i, m in enumerate(rows) for j in range(m)]
    pick = [0, 2, 3, 42, 43, 100, 172, 173, 232, 233, 234, 249]
    check_rows(out.float().cpu().numpy()[pick], qf[pick], refs, [places[i] for i in pick], hd ** -0.5, dtype)
    for i, m in enumerate(rows):
        alone = hs.Kv8Set([kvs[i]], n_heads=nh)
        part = torch.empty_like(q[:m])
        alone.attend(0, q[start[i]:start[i + 1]], part, i32([pos[i]]), i32([0, m]))
        assert torch.equal(part, out[start[i]:start[i + 1]])
        alone.close()
    # captured, on another stream, and beside a call on another set
    side, first = torch.cuda.Stream(), out.clone()
    start_d, pos_d = i32(start), i32(pos)
    twin, out2 = hs.Kv8Set(kvs[:1], n_heads=nh), torch.empty_like(q[:3])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        s.attend(0, q, out, pos_d, start_d, stream=side.cuda_stream)
    for _ in range(3):
        out.fill_(9.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        twin.attend(0, q[:3], out2, i32(pos[:1]), i32([0, 3]))
        torch.cuda.synchronize()
        assert torch.equal(out, first) and torch.equal(out2, first[:3])


def test_a_shared_chunk_keeps_non_finite_values_apart():
    """A NaN scale at one position of a split: rows before it do not see it, rows from it on are NaN."""
    rng = np.random.default_rng(8)
    kvs, refs = filled(rng, [9000], 2, 64, 1, 0, max_ctx=9100)
    s = hs.Kv8Set(kvs, n_heads=14)
    k, _ = rows_of(rng, 10, 2, 64, "f32")
    k[5] = float("nan")
    s.append(0, k, k, i32([9000]), i32([0, 10]))
    for dtype in ("f32", "f16", "bf16"):
        q, qf = rows_of(rng, 20, 14, 64, dtype)
        out = torch.empty_like(q)
        s.attend(0, q, out, i32([8990]), i32([0, 20]))
        assert bool(out[15:].isnan().all()) and not bool(out[:15].isnan().any())
        check_rows(out.float().cpu().numpy()[[0, 9]], qf[[0, 9]], refs, [(0, 8990), (0, 8999)], 0.125, dtype)


def test_offsets_past_32_bits():
    """A layer behind 4 GiB of others."""
    spec = hs.KvSpec(3, 8, 128, 1 << 20, 1)
    kv = hs.Kv.alloc8(spec, block=16)
    assert kv.bytes > 2 ** 32
    s = hs.Kv8Set([kv], n_heads=8)
    rng = np.random.default_rng(0)
    ref = Cache(8, 128, 64, 16)
    k, kf = rows_of(rng, 40, 8, 128, "f32")
    s.append(2, k, k, i32([0]), i32([0, 40]))
    ref.append(0, kf, kf)
    back = torch.empty_like(k)
    s.read(2, back, None, i32([0]), i32([0, 40]))
    assert torch.equal(back.cpu(), torch.from_numpy(ref.values(0, 0, 40)))
    out = torch.empty_like(k)
    s.attend(2, k, out, i32([0]), i32([0, 40]))
    check_rows(out.cpu().numpy()[[0, 39]], kf[[0, 39]], [ref], [(0, 0), (0, 39)], 128 ** -0.5, "f32")
    s.attend(2, k[:1], out[:1], i32([39]))
    check_rows(out.cpu().numpy()[:1], kf[:1], [ref], [(0, 39)], 128 ** -0.5, "f32")
    last = (1 << 20) - 1
    s.append(2, k[:1], k[:1], i32([last]))
    s.read(2, back[:1], None, i32([last]))
    assert torch.equal(back[:1].cpu(), torch.from_numpy(ref.values(0, 0, 1))[:1]) or bool((back[0] - k[0]).abs().max() < 0.05)
    s.check()


def test_a_rows_bits_do_not_depend_on_the_batch():
    rng = np.random.default_rng(21)
    lens = [900, 33, 2000, 512]
    kvs, _ = filled(rng, lens, 2, 64, 1, 0)
    both = hs.Kv8Set(kvs, n_heads=14)
    q, _ = rows_of(rng, 4, 14, 64, "f32")
    out = torch.empty_like(q)
    both.attend(0, q, out, i32([n - 1 for n in lens]))
    qc, _ = rows_of(rng, 160, 14, 64, "f32")
    outc = torch.empty_like(qc)
    both.attend(0, qc, outc, i32([n - 20 for n in lens[:1]] + [lens[1] - 20, lens[2] - 100, lens[3] - 20]),
                i32([0, 20, 40, 140, 160]))
    starts = [0, 20, 40, 140, 160]
    for i, n in enumerate(lens):
        s = hs.Kv8Set([kvs[i]], n_heads=14)
        one = torch.empty_like(q[:1])
        s.attend(0, q[i:i + 1], one, i32([n - 1]))
        assert torch.equal(one[0], out[i])
        m = starts[i + 1] - starts[i]
        part = torch.empty_like(qc[:m])
        s.attend(0, qc[starts[i]:starts[i + 1]], part, i32([n - m]), i32([0, m]))
        assert torch.equal(part, outc[starts[i]:starts[i + 1]])
        s.close()


def test_repeated_captured_and_side_stream_calls_agree():
    rng = np.random.default_rng(31)
    kvs, refs = filled(rng, [600, 77], 2, 128, 16, 0, max_ctx=700)
    s = hs.Kv8Set(kvs, n_heads=12)
    q, _ = rows_of(rng, 2, 12, 128, "bf16")
    k, kf = rows_of(rng, 2, 2, 128, "bf16")
    out = torch.empty_like(q)
    pos = i32([600, 77])
    s.append(0, k, k, pos)
    s.attend(0, q, out, pos)
    first = out.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out.zero_()
        s.append(0, k, k, pos, stream=side.cuda_stream)
        s.attend(0, q, out, pos, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(out, first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        s.append(0, k, k, pos, stream=side.cuda_stream)
        s.attend(0, q, out, pos, stream=side.cuda_stream)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first)
    # the same graph at other positions: the slots one and two positions further
    k2, _ = rows_of(rng, 2, 2, 128, "bf16")
    k.copy_(k2)
    pos.copy_(i32([601, 78]))
    graph.replay()
    torch.cuda.synchronize()
    want = torch.empty_like(q)
    s.attend(0, q, want, i32([601, 78]))
    assert torch.equal(out, want) and not torch.equal(out, first)


def test_refusals_on_the_gpu(tiny_gguf):
    spec = hs.KvSpec(2, 2, 64, 32, 0)
    a, b = hs.Kv.alloc8(spec), hs.Kv.alloc8(spec, block=16)
    c = hs.Kv.alloc8(hs.KvSpec(2, 2, 64, 33, 0))
    m = hs.Model.load(tiny_gguf, max_ctx=32)
    for kvs, heads in (([a, a], 2), ([a, b], 2), ([a, c], 2), ([m.kv()], 4), ([a], 3), ([a], 2 * 257)):
        with pytest.raises(hs.HotseatError) as e:
            hs.Kv8Set(kvs, n_heads=heads)
        assert e.value.code == hs.HS_E_ARG
    s = hs.Kv8Set([a], n_heads=4)
    none = hs.Kv8Set([a])
    q, k = torch.zeros(1, 4, 64, device="cuda"), torch.zeros(1, 2, 64, device="cuda")
    pos = i32([0])
    bad = [
        lambda: s.append(2, k, k, pos), lambda: s.read(2, k, k, pos), lambda: s.attend(2, q, torch.empty_like(q), pos),
        lambda: none.attend(0, torch.zeros(1, 0, 64, device="cuda"), torch.zeros(1, 0, 64, device="cuda"), pos),
        lambda: s.append(0, k.expand(2, 2, 64), k.expand(2, 2, 64), pos),  # two rows, one slot, no row_start
        lambda: s.read(0, k.expand(2, 2, 64), None, pos, i32([0, 2])),     # rows of an output overlap
        lambda: s.attend(0, q, torch.empty_like(q), pos, scale=0.0),
        lambda: s.attend(0, q, torch.empty_like(q), pos, scale=float("nan")),
        lambda: s.attend(0, q, torch.empty_like(q), pos, scale=float("inf")),
    ]
    for call in bad:
        with pytest.raises(hs.HotseatError) as e:
            call()
        assert e.value.code == hs.HS_E_ARG
    odd = [
        lambda: s.append(0, k.double(), k.double(), pos), lambda: s.append(0, k, k.half(), pos),
        lambda: s.append(0, k, k, pos.long()), lambda: s.append(0, k, k, i32([0, 0])), lambda: s.append(0, q, q, pos),
        lambda: s.append(0, k.cpu(), k.cpu(), pos), lambda: s.attend(0, k, k, pos),
        lambda: s.append(0, k, k, pos, row_start=i32([0])),
        lambda: s.append(0, torch.zeros(1, 2, 128, device="cuda")[..., ::2], torch.zeros(1, 2, 128, device="cuda")[..., ::2], pos),
    ]
    for call in odd:
        with pytest.raises(ValueError):
            call()
    s.append(0, k[:0], k[:0], pos, row_start=i32([0, 0]))  # no rows: nothing to do
    with pytest.raises(hs.HotseatError) as e:
        m.forward(m.kv8(), 1, 0, m.scratch())
    assert e.value.code == hs.HS_E_UNSUPPORTED
    with pytest.raises(hs.HotseatError) as e:
        a.copy_runs_to(b, [(0, 256)])
    assert e.value.code == hs.HS_E_ARG
