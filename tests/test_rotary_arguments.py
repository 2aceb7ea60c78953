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


@pytest.mark.parametrize('scaling', [
    {'rope_type': 'linear'}, {'rope_type': 'yarn', 'factor': None, 'original_max_position_embeddings': 4096},
    {'rope_type': 'llama3', 'factor': 8.0, 'original_max_position_embeddings': 8192},
    {'rope_type': 'llama3', 'factor': 8.0, 'original_max_position_embeddings': 8192, 'low_freq_factor': 1.0},
    {'rope_type': 'llama3', 'factor': 8.0, 'original_max_position_embeddings': 8192, 'low_freq_factor': 4.0, 'high_freq_factor': 4.0},
    {'rope_type': 'linear', 'factor': float('nan')}, {'rope_type': 'linear', 'factor': float('inf')}])
def test_entries_without_a_table_are_refused(scaling):
    """Missing keys, and values whose table would hold NaN or zeros."""
    with pytest.raises(ValueError):
        rotary_frequencies(64, 1e4, scaling)
