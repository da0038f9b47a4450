"""TokenReader's construction and refusals (CPU)."""

import pytest
import torch

from gaussian_splat_encoder.token_ops import RotaryAxes
from gaussian_splat_encoder.token_reader import TokenReader


def test_a_new_reader_has_zero_gates_and_the_usual_sizes():
    r = TokenReader(64, 40, RotaryAxes((8, 4, 4)), heads=4, kv_heads=2)
    assert r.head_dim == 16 and r.to_kv.out_features == 2 * 2 * 16 and r.fc1.out_features == 128
    assert not r.gate1.any() and not r.gate2.any() and torch.equal(r.norm1, torch.ones(64))
    assert sorted(n for n, _ in r.named_parameters() if "." not in n) == ["gate1", "gate2", "norm1", "norm2", "post1", "post2"]


@pytest.mark.parametrize("kw,what", [
    (dict(heads=4, kv_heads=3), "do not divide"), (dict(heads=0), "do not divide"), (dict(heads=5), "give head_dim"),
    (dict(heads=8), "RotaryAxes of 8 values"), (dict(axes=(8, 4)), "RotaryAxes")])
def test_wrong_sizes_are_refused(kw, what):
    kw = dict(dict(axes=RotaryAxes((8, 4))), **kw)
    with pytest.raises(ValueError, match=what):
        TokenReader(64, 40, **kw)


def test_cpu_tensors_are_refused():
    r = TokenReader(64, 40, RotaryAxes((8, 4)))
    with pytest.raises(RuntimeError, match="device tensors"):
        r(torch.zeros(1, 2, 64), torch.zeros(2, 2), torch.zeros(1, 3, 40), torch.zeros(3, 2))
