"""Arguments of rotary tables that mean something else than they did or are refused with a ValueError (no GPU: refusals come
before the device is asked for)."""
import pytest
import torch

from seedplane_amd.paged import Rotary, rotary_frequencies


def test_no_rotated_values_is_not_the_whole_head():
    for bad in (lambda: Rotary(64, rot_dim=0), lambda: Rotary.from_config({'head_dim': 64, 'partial_rotary_factor': 0.0}),
                lambda: Rotary.from_config({'head_dim': 64, 'rope_parameters': {'partial_rotary_factor': 0.0}}),
                lambda: Rotary.from_config({'head_dim': 64, 'partial_rotary_factor': 0.01})):
        with pytest.raises(ValueError, match='rot_dim'):
            bad()


def test_an_empty_rope_type_leaves_the_older_key_its_say():
    want = rotary_frequencies(64, 1e4, {'type': 'linear', 'factor': 2.0})[0]
    assert torch.equal(want, rotary_frequencies(64, 1e4)[0] / 2)
    assert torch.equal(rotary_frequencies(64, 1e4, {'rope_type': None, 'type': 'linear', 'factor': 2.0})[0], want)
