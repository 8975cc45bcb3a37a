"""The batched path over 8-bit regions: what it stores, its logits beside the
f32 cache's, prompts in passes, batches, live migration, the scoring command.

How far logits may be from the f32 cache's: a stored value is within half a
step of a block's or row's scale, step = max / 127; for 64 normal values
max is about 2.5 rms, so an rms error of 2.5 / 127 / sqrt(12) = 0.6%, on V
and, by the scores (of size about 1), on the weights: about 1% of an
attention output, of which the residual stream and two layers leave less than
2% in the logits. A scale over 16 positions and heads that share it: max about
3.5 rms, and up to twice the step where it grew: 4 times that. Bounds below:
5% and 15%, in the 2-norm."""
import numpy as np
import pytest

import hotseat_b200 as hs
from hotseat_b200 import ppl
from kv8_ref import Cache

from conftest import TINY

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def rows_f32(kv, layer, n):
    """K and V rows [n, nkv, hd] of an f32 region (token-major or head-major)."""
    s = kv.spec
    plane = s.max_ctx * s.n_kv_heads * s.head_dim
    f = kv.floats()[layer * 2 * plane:(layer + 1) * 2 * plane].reshape(2, plane)
    if s.layout == hs.TOKEN_MAJOR:
        return f.reshape(2, s.max_ctx, s.n_kv_heads, s.head_dim)[:, :n]
    return f.reshape(2, s.n_kv_heads, s.max_ctx, s.head_dim).transpose(0, 2, 1, 3)[:, :n]


def values8(kv, layer, n):
    s = hs.Kv8Set([kv])
    k = torch.empty(n, kv.spec.n_kv_heads, kv.spec.head_dim, device="cuda")
    v = torch.empty_like(k)
    s.read(layer, k, v, torch.zeros(1, dtype=torch.int32, device="cuda"),
           torch.tensor([0, n], dtype=torch.int32, device="cuda"))
    s.check()
    return k.cpu().numpy(), v.cpu().numpy()


def off(a, b):
    return float(np.linalg.norm(a.astype(np.float64) - b) / np.linalg.norm(b.astype(np.float64)))


@pytest.mark.parametrize("which, block, layout", [("tiny", 1, 0), ("tiny", 16, 1), ("tiny128", 1, 1), ("tiny128", 64, 0)])
def test_decode_steps(tiny_gguf, tiny128_gguf, which, block, layout):
    m = hs.Model.load(tiny_gguf if which == "tiny" else tiny128_gguf, max_ctx=96, numeric=hs.NUMERIC_TC)
    b8, b32 = hs.Batch(m, 3), hs.Batch(m, 3)
    kv8, kv32 = [m.kv8(layout, block) for _ in range(3)], [m.kv(layout) for _ in range(3)]
    rng = np.random.default_rng(1)
    c = m.cfg
    refs = [Cache(c.n_kv_heads, c.head_dim, 96, block) for _ in range(3)]
    for p in range(40):
        toks = rng.integers(0, c.vocab, 3)
        pos = [p, p, p]
        b8.forward(kv8, toks, pos)
        b32.forward(kv32, toks, pos)
        for i in range(3):
            assert off(b8.logits(i), b32.logits(i)) <= (0.05 if block == 1 else 0.15)
    # layer 0's rows depend on no attention: the f32 cache's, quantised
    for i in range(3):
        k, v = rows_f32(kv32[i], 0, 40)
        for p in range(40):
            refs[i].append(p, k[p:p + 1], v[p:p + 1])
        k8, v8 = values8(kv8[i], 0, 40)
        assert np.array_equal(k8, refs[i].values(0, 0, 40)) and np.array_equal(v8, refs[i].values(1, 0, 40))


def test_a_slots_bits_do_not_depend_on_its_batch(tiny_gguf):
    m = hs.Model.load(tiny_gguf, max_ctx=64, numeric=hs.NUMERIC_TC)
    b, one = hs.Batch(m, 70), hs.Batch(m, 1)
    kvs, alone = [m.kv8() for _ in range(70)], m.kv8()
    rng = np.random.default_rng(2)
    for p in range(12):
        toks = rng.integers(0, m.cfg.vocab, 70)
        b.forward(kvs, toks, [p] * 70)
        one.forward([alone], toks[17:18], [p])
        assert np.array_equal(b.logits(17), one.logits(0))
    assert kvs[17].hash(12) == alone.hash(12)


@pytest.mark.parametrize("block", [1, 32])
def test_prompts_in_passes(tiny_gguf, block):
    """A prompt in one pass and in several: the same layer-0 rows, logits as near as the cache's steps allow."""
    m = hs.Model.load(tiny_gguf, max_ctx=256, numeric=hs.NUMERIC_TC)
    rng = np.random.default_rng(3)
    prompt = rng.integers(0, m.cfg.vocab, 150)
    whole, pieces, f32 = m.kv8(block=block), m.kv8(block=block), m.kv()
    big, small, dec = hs.Batch(m, 192), hs.Batch(m, 64), hs.Batch(m, 1)
    big.prefill(whole, prompt)
    small.prefill(pieces, prompt[:70])
    small.prefill(pieces, prompt[70:], pos0=70)
    big.prefill(f32, prompt)
    logits = []
    for kv in (whole, pieces, f32):
        dec.forward([kv], [5], [150])
        logits.append(dec.logits(0))
    tol = 0.05 if block == 1 else 0.15
    assert off(logits[0], logits[2]) <= tol and off(logits[1], logits[2]) <= tol
    if block == 1:
        a, b = values8(whole, 0, 150), values8(pieces, 0, 150)
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])
        ref = Cache(m.cfg.n_kv_heads, m.cfg.head_dim, 256, 1)
        k, v = rows_f32(f32, 0, 150)
        ref.append(0, k, v)
        assert np.array_equal(a[0], ref.values(0, 0, 150)) and np.array_equal(a[1], ref.values(1, 0, 150))


@pytest.mark.parametrize("block", [1, 16])
def test_sequences_run_and_migrate(tiny_gguf, block):
    """Greedy sequences decoded on the device, one of them handed over midway by dirty pages."""
    m = hs.Model.load(tiny_gguf, max_ctx=128, numeric=hs.NUMERIC_TC)
    cfg = hs.SamplerCfg.default(temperature=0.0)
    rng = np.random.default_rng(4)
    prompts = [rng.integers(0, m.cfg.vocab, n).astype(np.uint32) for n in (9, 30)]

    def seqs():
        return [dict(tokens=p, prompt_len=len(p), max_tokens=60, cfg=cfg, rng=hs.Rng.seed(7)) for p in prompts]

    b = hs.Batch(m, 2)
    straight = [m.kv8(block=block) for _ in prompts]
    want = b.run_seqs(straight, seqs())
    src = [m.kv8(block=block) for _ in prompts]
    dst = m.kv8(block=block)
    half = b.run_seqs(src, seqs(), stop_at_filled=40)
    g = hs.Migration(src[0], dst, half[0][1].filled, len(half[0][0]), target_bytes=0)
    rest = [dict(tokens=t, prompt_len=s.prompt_len, max_tokens=s.max_tokens, cfg=cfg, rng=r, filled=s.filled, done=s.done,
                 done_reason=s.done_reason) for t, s, r in half]
    more = b.run_seqs(src, rest, stop_at_filled=50)
    assert g.round(more[0][1].filled, len(more[0][0])) in (True, False)
    rep = g.finish(more[0][1].filled, len(more[0][0]))
    assert rep["live_bytes"] > 0
    assert dst.hash(more[0][1].filled) == src[0].hash(more[0][1].filled)
    rest = [dict(tokens=t, prompt_len=s.prompt_len, max_tokens=s.max_tokens, cfg=cfg, rng=r, filled=s.filled, done=s.done,
                 done_reason=s.done_reason) for t, s, r in more]
    got = b.run_seqs([dst, src[1]], rest)
    for (t, s, _), (tw, sw, _) in zip(got, want):
        assert t.tolist() == tw.tolist() and s.filled == sw.filled
    assert dst.hash(got[0][1].filled) == straight[0].hash(want[0][1].filled)
    # a quarter of the f32 cache's bytes, and the scales
    f32 = m.kv()
    assert straight[0].bytes < 0.29 * f32.bytes


def test_formats_do_not_mix(tiny_gguf):
    m = hs.Model.load(tiny_gguf, max_ctx=64, numeric=hs.NUMERIC_TC)
    b = hs.Batch(m, 2)
    with pytest.raises(hs.HotseatError) as e:
        b.forward([m.kv8(), m.kv()], [1, 2], [0, 0])
    assert e.value.code == hs.HS_E_ARG
    with pytest.raises(hs.HotseatError) as e:
        b.forward([m.kv8(), m.kv8(block=16)], [1, 2], [0, 0])
    assert e.value.code == hs.HS_E_ARG
    for src, dst in ((m.kv8(), m.kv()), (m.kv8(), m.kv8(block=16)), (m.kv(), m.kv8())):
        with pytest.raises(hs.HotseatError) as e:
            hs.Migration(src, dst, 0, 1)
        assert e.value.code == hs.HS_E_STATE and "format" in str(e.value)
    # one batch decodes over either, in turn
    a, c = m.kv8(), m.kv()
    b.forward([a], [3], [0])
    x = b.logits(0)
    b.forward([c], [3], [0])
    y = b.logits(0)
    assert off(x, y) <= 0.05
    b.forward([m.kv8()], [3], [0])
    assert np.array_equal(b.logits(0), x)


def test_scoring_with_an_8_bit_cache_and_detail(tiny_gguf):
    m = hs.Model.load(tiny_gguf, max_ctx=32, numeric=hs.NUMERIC_TC)
    ids = [int(t) for t in np.random.default_rng(17).integers(0, TINY["vocab"], size=3 * 32)]
    plain = ppl.score(m, ids, 32)
    more = ppl.score(m, ids, 32, detail=True)
    assert more["mean_nll"] == plain["mean_nll"] and more["scored"] == plain["scored"]
    assert 0 < more["mean_entropy"] <= np.log(TINY["vocab"]) + 1e-5 and 0 <= more["top1"] <= more["top5"] <= 1
    # a score moves by at most twice the logits' largest move: 5% of their norm, were it all in one
    eight = ppl.score(m, ids, 32, detail=True, kv8=1)
    assert eight["scored"] == plain["scored"] and abs(eight["mean_nll"] - plain["mean_nll"]) <= 0.5
    f = hs.Model.load(tiny_gguf, max_ctx=32, numeric=hs.NUMERIC_FAST)
    d = ppl.score(f, ids, 32, detail=True)
    assert abs(d["mean_entropy"] - more["mean_entropy"]) <= 2e-2
