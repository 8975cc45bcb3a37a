"""What calls on 8-bit regions and logits refuse and take: places, strides and
shapes of tensors."""
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
