"""Device memory that the batched path takes over 8-bit regions."""
import numpy as np
import pytest

import hotseat_b200 as hs

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def free():
    torch.cuda.synchronize()
    return torch.cuda.mem_get_info()[0]


def test_a_prefill_over_8_bit_regions_takes_no_workspace_of_other_paths(tiny_gguf):
    """256 slots of 32,768 positions: the join records of single rows are 256 x 2 heads x 16 clusters x 2,560 bytes,
    20 MiB, and the f32 prefill's segment records as much again. A prefill needs neither; the first decode step
    takes the former."""
    m = hs.Model.load(tiny_gguf, max_ctx=32768, numeric=hs.NUMERIC_TC)
    b, kv = hs.Batch(m, 256), m.kv8()
    warm = hs.Batch(m, 64)  # the library's kernels and graphs are there
    warm.prefill(m.kv8(), np.arange(64) % m.cfg.vocab)
    warm.forward([m.kv8()], [1], [0])
    prompt = np.arange(200) % m.cfg.vocab
    before = free()
    b.prefill(kv, prompt)
    after = free()
    assert before - after < 16 << 20
    b.forward([kv], [5], [200])
    first = b.logits(0)
    assert after - free() >= 20 << 20
    b.prefill(kv, prompt)  # again, either way, on the same buffers
    b.forward([kv], [5], [200])
    assert np.array_equal(b.logits(0), first)
    one = hs.Batch(m, 1)
    one.forward([kv], [5], [200])
    assert np.array_equal(one.logits(0), first)
