"""Construction and refusals of CellReader and of the encoder's options (CPU; no kernel runs)."""

import pytest
import torch

from gaussian_splat_encoder import efficient_encoder as EE
from gaussian_splat_encoder.cell_reader import CellReader
from gaussian_splat_encoder.checkpoint import encoder_kwargs


def test_options_are_off_by_default_and_add_no_parameters():
    a = EE.EfficientGaussianEncoder(d_feature=32, variant="adaptive", fine_stride=4)
    b = EE.EfficientGaussianEncoder(d_feature=32, variant="adaptive", fine_stride=4, channels_last=True)
    assert list(a.state_dict()) == list(b.state_dict())
    c = EE.EfficientGaussianEncoder(d_feature=32, variant="adaptive", fine_stride=4, fine_reader_heads=4)
    extra = set(c.state_dict()) - set(a.state_dict())
    assert extra and all(k.startswith("fine_reader.") for k in extra)
    kw = encoder_kwargs({"d_feature": 32, "variant": "adaptive", "fine_stride": 4, "fine_reader_heads": 4})
    assert list(EE.EfficientGaussianEncoder(**kw).state_dict()) == list(c.state_dict())


@pytest.mark.parametrize("kw", [dict(norm_type="instance", channels_last=True), dict(variant="free", fine_reader_heads=2)])
def test_encoder_refuses(kw):
    with pytest.raises(ValueError):
        EE.EfficientGaussianEncoder(d_feature=32, **kw)


@pytest.mark.parametrize("a,kw", [((32, 16), dict(heads=3)), ((32, 16), dict(heads=4, kv_heads=3)), ((32, 16), dict(heads=0)),
                                  ((30, 16), dict(heads=2, groups=8))])
def test_reader_refuses(a, kw):
    with pytest.raises(ValueError):
        CellReader(*a, **kw)


def test_reader_needs_states():
    with pytest.raises(ValueError, match="states or kv"):
        CellReader(32, 16)(torch.zeros(1, 4, 32))


def test_host_tensors_are_refused():
    with pytest.raises(RuntimeError, match="device tensors"):
        CellReader(32, 16)(torch.zeros(1, 4, 32), torch.zeros(1, 3, 16))
    with pytest.raises(RuntimeError, match="device tensors"):
        EE.EfficientGaussianEncoder(d_feature=32, channels_last=True)(torch.zeros(1, 3, 32, 32))
