"""The 8-bit KV cache without a GPU: live ranges, refusals, and the
restatement that the GPU tests compare with."""
import ctypes as C

import numpy as np
import pytest

import hotseat_b200 as hs
from kv8_ref import Cache, codes_of, need_of


def test_live_ranges_hold_every_row_and_scale_once():
    for layout in (0, 1):
        for block in (1, 16, 128):
            s = hs.KvSpec(3, 2, 64, 1000, layout)
            pad = lambda n: -(-n // 256) * 256  # noqa: E731
            plane, splane = pad(1000 * 2 * 64), pad(-(-1000 // block) * 2 * 4)
            for a, b in ((0, 0), (5, 5), (7, 3), (0, 1), (0, 1000), (37, 300), (999, 1000)):
                got = hs.live_ranges_between8(s, block, a, b)
                if b <= a:
                    assert got == []
                    continue
                a0 = a // block * block
                nb = -(-b // block) - a0 // block
                assert sum(n for _, n in got) == 3 * 2 * ((b - a0) * 2 * 64 + nb * 2 * 4)
                ends = [(o, o + n) for o, n in got]
                assert all(x[1] <= y[0] for x, y in zip(ends, ends[1:]))
                assert ends[-1][1] <= 3 * 2 * (plane + splane)
                assert len(got) == 3 * 4 * (1 if layout == 0 else 2)


def test_a_block_that_is_no_power_of_two_has_no_ranges():
    assert hs.live_ranges_between8(hs.KvSpec(1, 1, 64, 10, 0), 3, 0, 5) == []
    assert hs.live_ranges_between8(hs.KvSpec(1, 1, 64, 10, 0), 0, 0, 5) == []


@pytest.mark.parametrize("spec, block, code", [
    ((1, 1, 96, 8, 0), 1, hs.HS_E_UNSUPPORTED), ((1, 1, 64, 8, 0), 8, hs.HS_E_UNSUPPORTED),
    ((1, 1, 64, 8, 0), 256, hs.HS_E_UNSUPPORTED), ((1, 1, 64, 8, 2), 1, hs.HS_E_ARG), ((0, 1, 64, 8, 0), 1, hs.HS_E_ARG),
    ((1, 0, 64, 8, 0), 1, hs.HS_E_ARG), ((1, 1, 64, 0, 0), 1, hs.HS_E_ARG), ((1, 1, 64, 8, 0), 0, hs.HS_E_ARG),
])
def test_shapes_refused_before_any_device_call(spec, block, code):
    with pytest.raises(hs.HotseatError) as e:
        hs.Kv.alloc8(hs.KvSpec(*spec), block=block)
    assert e.value.code == code


def test_page_sizes_refused():
    for page in (0, 100, 128, 5000):
        with pytest.raises(hs.HotseatError) as e:
            hs.Kv.alloc8(hs.KvSpec(1, 1, 64, 8, 0), page_size=page)
        assert e.value.code == hs.HS_E_ARG


def test_null_arguments():
    lib, h = hs.lib(), C.c_void_p()
    assert lib.hs_kv8_alloc(0, None, 1, 4096, 0, C.byref(h)) == hs.HS_E_ARG
    assert lib.hs_kv8_alloc_model(None, 0, 1, 4096, C.byref(h)) == hs.HS_E_ARG
    assert lib.hs_kv8_open_ipc(None, None, 0, 1, 4096, C.byref(h)) == hs.HS_E_ARG
    assert lib.hs_kv8_block(None, None) == hs.HS_E_ARG
    assert lib.hs_kv8_set_new(None, 1, 0, C.byref(h)) == hs.HS_E_ARG
    assert lib.hs_kv8_set_new((C.c_void_p * 1)(None), 1, 0, C.byref(h)) == hs.HS_E_ARG
    assert lib.hs_kv8_set_new((C.c_void_p * 1)(None), 0, 0, C.byref(h)) == hs.HS_E_ARG
    assert lib.hs_kv8_set_check(None, None) == hs.HS_E_ARG
    assert lib.hs_kv8_append(None, 0, 1, None, None, None, None, 0, 64, 64, None) == hs.HS_E_ARG
    assert lib.hs_kv8_read(None, 0, 1, None, None, None, None, 0, 64, 64, None) == hs.HS_E_ARG
    assert lib.hs_kv8_attend(None, 0, 1, None, None, None, 64, 64, None, 64, 64, 0, 1.0, None) == hs.HS_E_ARG
    lib.hs_kv8_set_free(None)


def test_logprobs_refusals():
    lib, p = hs.lib(), C.c_void_p(4096)  # a pointer that no refused call follows
    call = lambda logits=p, dtype=0, rows=1, vocab=10, ids=p, top=0, logp=p, rank=None, tid=None, tlp=None: (  # noqa: E731
        lib.hs_logprobs(0, logits, dtype, vocab, rows, vocab, ids, top, logp, None, rank, tid, tlp, None))
    assert call(vocab=0) == hs.HS_E_ARG
    assert call(dtype=3) == hs.HS_E_ARG
    assert call(logits=None) == hs.HS_E_ARG
    assert call(logits=C.c_void_p(4097)) == hs.HS_E_ARG
    assert call(ids=None) == hs.HS_E_ARG
    assert call(ids=None, logp=None, rank=p) == hs.HS_E_ARG
    assert call(top=65, vocab=100, tid=p) == hs.HS_E_ARG
    assert call(top=11, tid=p) == hs.HS_E_ARG
    assert call(top=0, tid=p) == hs.HS_E_ARG
    assert call(top=0, tlp=p) == hs.HS_E_ARG
    assert call(rows=0) == hs.HS_OK  # nothing to do, no device needed
    assert lib.hs_scratch_logprobs(None, 0, 0, None, None, None, None, None) == hs.HS_E_ARG
    assert lib.hs_batch_logprobs(None, None, 0, 0, None, None, None, None, None) == hs.HS_E_ARG


def test_restated_quantiser():
    x = np.array([[0.5, -1.0, 0.25, 127.0]], np.float32)
    s = need_of(x)
    assert s == np.float32(1.0)
    assert codes_of(x, s).tolist() == [[0, -1, 0, 127]]  # 0.5 ties to even
    assert codes_of(np.array([1.5, 2.5, -1.5], np.float32), np.float32(1)).tolist() == [2, 2, -2]
    assert np.isnan(need_of(np.array([1.0, np.inf]))) and np.isnan(need_of(np.array([1.0, np.nan])))
    assert need_of(np.zeros(4)) == 0 and need_of(np.full(4, 1e-40, np.float32)) == 0


@pytest.mark.parametrize("block", [16, 64])
def test_values_stay_within_a_step_however_a_block_fills(block):
    rng = np.random.default_rng(block)
    c = Cache(1, 64, 128, block)
    x = (rng.standard_normal((100, 1, 64)) * np.exp(rng.uniform(-2, 2, (100, 1, 1)))).astype(np.float32)
    for p in range(100):
        c.append(p, x[p:p + 1], x[p:p + 1])
    steps = c.scales[0][np.arange(100) // block]
    assert np.all(np.abs(c.values(0, 0, 100).astype(np.float64) - x) <= steps[:, :, None] * (1 + 2 ** -20))
    whole = Cache(1, 64, 128, block)
    whole.append(0, x, x)
    steps = whole.scales[0][np.arange(100) // block]
    assert np.all(np.abs(whole.values(0, 0, 100).astype(np.float64) - x) <= steps[:, :, None] * (0.5 + 2 ** -16))


@pytest.mark.parametrize("spec, block", [((1 << 20, 4096, 128, 1 << 30, 0), 1), ((1 << 31, 4096, 128, 1 << 30, 1), 16),
                                         ((0xFFFFFFFF, 1, 64, 1 << 30, 0), 128)])
def test_regions_whose_bytes_pass_64_bits_are_refused(spec, block):
    """2^20 layers of 2^50 + 2^45 bytes are 0 modulo 2^64: a region of no bytes, with layers behind it."""
    with pytest.raises(hs.HotseatError) as e:
        hs.Kv.alloc8(hs.KvSpec(*spec), block=block)
    assert e.value.code == hs.HS_E_UNSUPPORTED


def test_live_ranges_of_the_longest_context():
    s = hs.KvSpec(1, 2, 64, 0xFFFFFFFF, 1)
    got = hs.live_ranges_between8(s, 128, 0, 1)
    plane = -(-0xFFFFFFFF * 2 * 64 // 256) * 256
    assert got[4:6] == [(2 * plane, 4), (2 * plane + 4 * (1 << 25), 4)]  # the second head's scales behind the first's
