"""Refusals and bookkeeping of the token operators on the host (CPU; no kernel runs)."""

import pytest
import torch

from gaussian_splat_encoder import token_ops as F
from test_token_args import cache, ints, t

AX = F.RotaryAxes((8, 4))


@pytest.fixture
def no_launch(monkeypatch):
    """The names of what would be launched."""
    names = []
    monkeypatch.setattr(F, "_launch", lambda x, name, *args: names.append(name))
    return names


def calls(positions, c=None):
    c = cache() if c is None else c
    return (lambda: F.cache_append(c, ints(1, 2), ints(1), t(1, 1, 2, 16), t(1, 1, 2, 16), positions=positions, axes=AX),
            lambda: F.cached_attention(t(1, 1, 2, 16), c, ints(1, 2), ints(1), positions=positions, axes=AX))


def test_the_cache_has_no_gradients_of_positions(no_launch):
    """Splat centres that learn: their gradient would be dropped without a word."""
    learnt = t(1, 1, 2).requires_grad_(True)
    for call in calls(learnt):
        with pytest.raises(NotImplementedError, match="inference"):
            call()
        with torch.no_grad():
            call()
    for call in calls(learnt.detach()):
        call()
    assert len(no_launch) == 4
    with torch.autograd.forward_ad.dual_level():
        for call in calls(torch.autograd.forward_ad.make_dual(t(1, 1, 2), t(1, 1, 2))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def test_pages_that_came_to_require_a_gradient_are_refused(no_launch):
    c = cache()
    c.v.requires_grad_(True)
    for call in calls(t(1, 1, 2), c):
        with pytest.raises(NotImplementedError, match="inference"):
            call()
    assert not no_launch


def test_an_append_counts_as_a_write(no_launch):
    """Autograd knows of writes by its tensors' version counters; views of a page share them."""
    for c in (cache(), cache(masked=True)):
        page = c.k[0]
        before = [x._version for x in (c.k, c.v, page)] + ([] if c.live is None else [c.live._version])
        read = calls(t(1, 1, 2), c)
        read[1]()
        now = lambda: [x._version for x in (c.k, c.v, page)] + ([] if c.live is None else [c.live._version])  # noqa: E731
        assert now() == before
        read[0]()
        assert all(a > b for a, b in zip(now(), before))
        after = now()
        F.cache_append(c, ints(1, 2), ints(1), t(1, 0, 2, 16), t(1, 0, 2, 16))      # writes nothing
        assert now() == after and no_launch.count("splat_cache_append") == 1
        no_launch.clear()
    with torch.inference_mode():        # tensors without counters
        c = cache()
        calls(t(1, 1, 2), c)[0]()
    assert no_launch == ["splat_cache_append"]


@pytest.mark.parametrize("kw", [dict(dims=(64,), base=1e-320), dict(dims=(64,), base=1e-300, scale=1e300),
                                dict(dims=(4,), scale=1e300), dict(dims=(4, 4), scale=(1.0, -3.5e38))])
def test_rates_past_float32_are_refused(kw):
    """A position's product with them would pass 64 bits, its gradient float32."""
    with pytest.raises(ValueError, match="rates"):
        F.RotaryAxes(**kw)
    F.RotaryAxes((4,), scale=-3.4e38, base=1.0)


@pytest.mark.parametrize("H,Hk,D,n", [(4, 4, 64, 300), (8, 2, 128, 129), (32, 1, 96, 61)])
def test_one_bfloat16_value_for_two_would_show(H, Hk, D, n):
    """What test_gpu_token_edges allows a bfloat16 attention (1.05 of the exact result's own rounding) is passed where a
    probability or a turned query loses its second value: planted in the float64 attention."""
    import _token_ref as R
    from _feature_ref import rel
    b = torch.bfloat16
    g = torch.Generator().manual_seed(1)
    q, k, v = ((torch.randn(12, *s, D, generator=g) * f).to(b).double()
               for s, f in (((H,), 1.3), ((n, Hk), 1.3), ((n, Hk), 1.0)))
    k, v = k.repeat_interleave(H // Hk, 2), v.repeat_interleave(H // Hk, 2)
    q = R.rotary(q[:, None], torch.full((12, 1, 1), 12345.0, dtype=torch.float64), F.RotaryAxes((D,)))[:, 0]

    def attend(q, lose):
        s = (q[:, None] * k).sum(-1) * D ** -0.5
        w = torch.exp(s - s.amax(1, keepdim=True))
        return ((w.to(b).double() if lose else w)[..., None] * v).sum(1) / w.sum(1)[..., None]

    want = attend(q, False)
    own = rel(want.to(b), want)
    assert rel(attend(q, True).to(b), want) > 1.1 * own
    assert rel(attend(q.to(b).double(), False).to(b), want) > 1.5 * own


def test_an_append_into_expanded_pages_is_refused(no_launch):
    """Tokens that share memory may be read, but a call would write many of them to one place."""
    one = t(1, 8, 2, 16)
    for c in (F.PagedCache(one.expand(4, 8, 2, 16), t(4, 8, 2, 16)),
              F.PagedCache(t(4, 8, 2, 16), t(4, 1, 2, 16).expand(4, 8, 2, 16)),
              F.PagedCache(t(4, 8, 2, 16), t(4, 8, 2, 16), t(4, 1, dtype=torch.bool).expand(4, 8))):
        append, read = calls(t(1, 1, 2), c)
        with pytest.raises(ValueError, match="share memory"):
            append()
        read()
    calls(t(1, 1, 2), F.PagedCache(one.expand(1, 8, 2, 16), one))[0]()      # one page: nothing is shared
    assert no_launch == ["splat_cached_attention"] * 3 + ["splat_cache_append"]
