"""What calls on 8-bit regions and logits refuse and take: places, strides and
shapes of tensors."""
import pytest

import hotseat_b200 as hs
from test_gpu_kv8 import i32

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
