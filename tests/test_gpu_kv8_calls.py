"""What calls on 8-bit regions and logits refuse and take: places, strides and
shapes of tensors."""
import numpy as np
import pytest

import hotseat_b200 as hs
from kv8_ref import Cache
from test_gpu_kv8 import i32, raw, rows_of, same

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


class Elsewhere:
    """A tensor that says it lies on the next GPU."""

    def __init__(self, t):
        self.t = t

    def get_device(self):
        return self.t.get_device() + 1

    def __getattr__(self, name):
        return getattr(self.t, name)


def test_tensors_of_another_gpu_than_the_regions_are_refused():
    s = hs.Kv8Set([hs.Kv.alloc8(hs.KvSpec(1, 2, 64, 32, 0))], n_heads=4)
    k, q, pos = torch.ones(1, 2, 64, device="cuda"), torch.ones(1, 4, 64, device="cuda"), i32([0])
    away = Elsewhere
    for call in (lambda: s.append(0, away(k), away(k), away(pos)), lambda: s.read(0, away(k), away(k), away(pos)),
                 lambda: s.attend(0, away(q), away(torch.empty_like(q)), away(pos)), lambda: s.append(0, k, k, away(pos)),
                 lambda: s.append(0, k, away(k), pos), lambda: s.attend(0, q, away(torch.empty_like(q)), pos)):
        with pytest.raises(ValueError):
            call()
    s.append(0, k, k, pos)
    s.check()


@pytest.mark.parametrize("nkv, m", [(1, 5), (2, 1), (1, 1)])
def test_strides_of_single_rows_and_heads_do_not_count(nkv, m):
    """K a slice of a fused row, V on its own: alike where there is more than one row or head."""
    rng = np.random.default_rng(nkv + m)
    kv, ref = hs.Kv.alloc8(hs.KvSpec(1, nkv, 64, 32, 0)), Cache(nkv, 64, 32, 1)
    s = hs.Kv8Set([kv])
    wide, wf = rows_of(rng, m, 3 * nkv, 64, "f32")
    k = wide[:, :nkv] if m == 1 else torch.as_strided(wide, (m, 1, 64), (3 * 64, 640, 1))
    v = torch.as_strided(rows_of(rng, 3 * m, nkv, 64, "f32")[0], (m, nkv, 64), (192 if m > 1 else 77, 64, 1))
    s.append(0, k, v, i32([0]), i32([0, m]))
    ref.append(0, k.cpu().numpy(), v.cpu().numpy())
    same(kv, ref)
    out = torch.zeros(m, nkv, 64, device="cuda")
    s.read(0, torch.as_strided(out, out.shape, (64 * nkv if m > 1 else 11, 64 if nkv > 1 else 3, 1)),
           torch.zeros_like(out), i32([0]), i32([0, m]))
    assert torch.equal(out.cpu(), torch.from_numpy(ref.values(0, 0, m)))
    assert raw(kv)[0].shape[1] == 32
    with pytest.raises(ValueError):  # strides that do count
        s.append(0, torch.zeros(2, nkv, 128, device="cuda")[..., :64], torch.zeros(2, nkv, 64, device="cuda"), i32([0]), i32([0, 2]))


def test_outputs_of_other_shapes_are_refused():
    x, ids = torch.zeros(3, 50, device="cuda"), i32([1, 2, 3])
    f, n = torch.zeros(3, device="cuda"), torch.zeros(3, 2, device="cuda")
    for kw in (dict(top_logp=f), dict(top_logp=n[:2]), dict(top_logp=n[None]), dict(top_ids=n), dict(top_ids=ids),
               dict(top_ids=torch.zeros(3, 4, dtype=torch.int32, device="cuda"), top_logp=n), dict(logp=f[:2], ids=ids),
               dict(logp=n, ids=ids), dict(entropy=f.half()), dict(rank=f, ids=ids), dict(logp=f, ids=ids.long())):
        with pytest.raises(ValueError):
            hs.logprobs(x, **kw)


@pytest.mark.parametrize("block, layout", [(1, 0), (16, 1), (64, 0)])
def test_going_back(block, layout):
    """Rows taken back and appended anew, in the middle of a block and at its beginning."""
    rng = np.random.default_rng(block)
    spec = hs.KvSpec(1, 2, 64, 200, layout)
    kv, ref, fresh = hs.Kv.alloc8(spec, block=block), Cache(2, 64, 200, block), Cache(2, 64, 200, block)
    s = hs.Kv8Set([kv])
    x = (rng.standard_normal((200, 2, 64)) * np.exp(rng.uniform(-1, 1, (200, 1, 1)))).astype(np.float32)
    steps = np.zeros((200, 2), np.float32)  # the largest scale that each row has stood under

    def add(pos, rows):
        t = torch.from_numpy(rows).cuda()
        s.append(0, t, t, i32([pos]), i32([0, len(rows)]))
        ref.append(pos, rows, rows)
        now = ref.scales[0][np.arange(200) // block]
        steps[:] = np.maximum(steps, now)

    def values(n):
        k = torch.empty(n, 2, 64, device="cuda")
        s.read(0, k, None, i32([0]), i32([0, n]))
        return k.cpu().numpy()

    add(0, x[:150])
    held = values(150)
    big = 8 * x[:40]
    add(100, big)  # in a block for 16 and 64; the rows before it stay within a step of its scale
    got = values(140)
    assert np.array_equal(got, ref.values(0, 0, 140))
    assert np.array_equal(got[:100 // block * block], held[:100 // block * block])
    assert np.all(np.abs(got[:100].astype(np.float64) - x[:100]) <= steps[:100, :, None] * (1 + 2 ** -20))
    assert np.all(np.abs(got[100:].astype(np.float64) - big) <= steps[100:140, :, None] * (1 + 2 ** -20))
    if block == 1:
        assert np.array_equal(values(150)[140:], held[140:])  # rows behind stay
    # taken back to the beginning of a block: a fresh sequence's bytes
    back = 64
    add(back, x[back:150])
    fresh.append(0, x[:back], x[:back])
    fresh.append(back, x[back:150], x[back:150])
    codes, scales = raw(kv)
    nb = -(-150 // block)
    assert np.array_equal(scales[:, :nb], fresh.scales[:, :nb]) and np.array_equal(codes[:, :150], fresh.codes[:, :150])
    # a row that is not finite, taken back: its block stays NaN where it held older rows
    bad = np.full((1, 2, 64), np.nan, np.float32)
    add(70, bad)
    add(70, x[70:72])
    got = values(72)
    assert np.isnan(got[70]).all() == (block > 1) and np.array_equal(np.isnan(got[64:70]).all(), block > 1)
    add(64, x[64:72])
    assert not np.isnan(values(72)).any()


@pytest.mark.parametrize("block", [1, 16])
def test_the_last_position_behind_4_gib(block):
    """A row of its own there, read into other values, and found at its own bytes only."""
    n = 1 << 20
    spec = hs.KvSpec(3, 8, 128, n, 1)
    kv = hs.Kv.alloc8(spec, block=block)
    assert kv.bytes > 2 ** 32
    s = hs.Kv8Set([kv], n_heads=8)
    rng = np.random.default_rng(block)
    k, kf = rows_of(rng, 3, 8, 128, "f32")
    ref = Cache(8, 128, block, block)
    ref.append(block - 1, kf[2:], kf[2:])  # the region's last block, of which it is the last row
    s.append(2, k[:2], k[:2], i32([0]), i32([0, 2]))
    first = torch.full_like(k[:2], 5.0)
    s.read(2, first, None, i32([0]), i32([0, 2]))
    s.append(2, k[2:], k[2:], i32([n - 1]))
    for which in range(2):
        back = torch.full_like(k[:1], 5.0)
        s.read(2, *((back, None) if which == 0 else (None, back)), i32([n - 1]))
        assert torch.equal(back.cpu(), torch.from_numpy(ref.values(which, block - 1, block)))
    again = torch.full_like(k[:2], 5.0)
    s.read(2, again, None, i32([0]), i32([0, 2]))
    assert torch.equal(first, again)
    # the code row of K's last head at the plane's end, of V's one plane on
    plane = n * 8 * 128
    at = 2 * (kv.bytes // 3)
    for which in range(2):
        row = kv.read(at + which * plane + plane - 128, 128).view(np.int8)
        assert np.array_equal(row, ref.codes[which, block - 1, 7]) and row.any()
    s.check()


@pytest.mark.parametrize("block", [1, 16])
def test_the_rounds_of_a_hand_over(tiny_gguf, block):
    """What each round sends: the rows since the one before, from the start of the block that they continue."""
    m = hs.Model.load(tiny_gguf, max_ctx=256, numeric=hs.NUMERIC_TC)
    src, dst, b = m.kv8(block=block, page_size=256), m.kv8(block=block, page_size=256), hs.Batch(m, 64)
    b.prefill(src, np.arange(100) % m.cfg.vocab)
    g = hs.Migration(src, dst, 100, 101, target_bytes=0)
    for p in range(100, 110):
        b.forward([src], [p], [p])
    assert g.round(110, 111) is True  # smaller than the whole, above the target of 0
    assert g.round(110, 111) is False  # nothing was written since
    for p in range(110, 113):
        b.forward([src], [p], [p])
    rep = g.finish(113, 114)
    assert [r["index"] for r in rep["rounds"]] == [0, 1] and rep["converged"] == 1
    assert rep["stop_reason"] == "nothing left to send"
    sent = lambda a, z: sum(n for _, n in hs.live_ranges_between8(m.kv_spec(), block, a, z))  # noqa: E731
    assert rep["rounds"][0]["bytes"] == sent(0, 101)
    # pages that hold the ten rows, clipped to the live ranges from their block's start on
    assert 10 * 2 * 2 * m.cfg.n_layers * 64 <= rep["rounds"][1]["bytes"] <= sent(100, 111)
    assert 0 < rep["final_bytes"] <= sent(110, 113) and rep["live_bytes"] == sent(0, 113)
    assert dst.hash(113) == src.hash(113)
