"""CPU tests of ``Rotary.from_config`` over the shapes a config's rope parameters take."""

from types import SimpleNamespace

import pytest


def test_parameters_for_each_kind_of_layer_are_refused():
    """Their theta would silently be the default one."""
    from turbopress_b200.rotary import Rotary
    kinds = dict(sliding_attention=dict(rope_type="default", rope_theta=10000.0),
                 full_attention=dict(rope_type="linear", factor=8.0, rope_theta=1e6))
    base = dict(head_dim=128, hidden_size=1024, num_attention_heads=8)
    for p in (kinds, {**kinds, "rope_type": "default", "rope_theta": None}):
        with pytest.raises(ValueError, match="each kind of layer"):
            Rotary.from_config(SimpleNamespace(**base, rope_parameters=p), device="cpu")
    for p in kinds.values():  # as the message says
        r = Rotary(128, theta=p["rope_theta"], scaling=p, device="cpu")
        assert abs(float(r.inv_freq[-1]) * p["rope_theta"] ** (126 / 128) * p.get("factor", 1.0) - 1) < 1e-5


def test_configs_without_scaling():
    from turbopress_b200.rotary import Rotary
    base = dict(head_dim=None, hidden_size=1024, num_attention_heads=8)
    for extra in (dict(), dict(rope_parameters=None), dict(rope_scaling=None, rope_theta=10000.0),
                  dict(rope_parameters=dict(rope_type="default", rope_theta=10000.0))):
        r = Rotary.from_config(SimpleNamespace(**base, **extra), device="cpu")
        assert r.rot_dim == 128 and abs(float(r.inv_freq[1]) * 10000.0 ** (1 / 64) - 1) < 1e-6
