"""Rotary frequencies for scaled contexts (host code): the published forms written out, and transformers' own tables."""
import math

import pytest
import torch

from seedplane_amd.paged import rotary_frequencies


def _published(rot, theta, s, length=None):
    """The forms from their papers, one pair at a time: position interpolation, NTK by length, YaRN (by wavelengths), llama3."""
    out = []
    kind, f, L = s['rope_type'], s['factor'], s.get('original_max_position_embeddings')
    for j in range(rot // 2):
        inv = theta ** (-2.0 * j / rot)
        wave = 2 * math.pi / inv
        if kind == 'linear':
            inv /= f
        elif kind == 'dynamic':
            n = max(length or L, L)
            inv = (theta * (f * n / L - (f - 1)) ** (rot / (rot - 2))) ** (-2.0 * j / rot)
        elif kind == 'llama3':
            if wave > L / s['low_freq_factor']:
                inv /= f
            elif wave >= L / s['high_freq_factor']:
                t = (L / wave - s['low_freq_factor']) / (s['high_freq_factor'] - s['low_freq_factor'])
                inv = (1 - t) * inv / f + t * inv
        else:
            at = lambda turns: rot * math.log(L / (turns * 2 * math.pi)) / (2 * math.log(theta))
            lo, hi = max(0, math.floor(at(s.get('beta_fast', 32)))), min(rot - 1, math.ceil(at(s.get('beta_slow', 1))))
            ramp = min(1.0, max(0.0, (j - lo) / max(hi - lo, 1e-3)))
            inv = inv / f * ramp + inv * (1 - ramp)
        out.append(inv)
    return torch.tensor(out, dtype=torch.float64)


SCALINGS = [
    ({'rope_type': 'linear', 'factor': 4.0}, None),
    ({'rope_type': 'dynamic', 'factor': 2.0, 'original_max_position_embeddings': 2048}, None),
    ({'rope_type': 'dynamic', 'factor': 2.0, 'original_max_position_embeddings': 2048}, 10000),
    ({'rope_type': 'yarn', 'factor': 4.0, 'original_max_position_embeddings': 32768}, None),
    ({'rope_type': 'yarn', 'factor': 2.5, 'original_max_position_embeddings': 4096, 'beta_fast': 16, 'beta_slow': 2}, None),
    ({'rope_type': 'llama3', 'factor': 8.0, 'low_freq_factor': 1.0, 'high_freq_factor': 4.0,
      'original_max_position_embeddings': 8192}, None),
]


@pytest.mark.parametrize('scaling,length', SCALINGS)
@pytest.mark.parametrize('rot,theta', [(128, 1e6), (64, 1e4), (32, 5e5)])
def test_scaled_tables(rot, theta, scaling, length):
    inv, factor = rotary_frequencies(rot, theta, scaling, length)
    assert inv.dtype == torch.float64 and inv.shape == (rot // 2,)
    want = _published(rot, theta, scaling, length)
    # a handful of 64-bit roundings and a power: 1e-12 of each value
    assert float(((inv - want) / want).abs().max()) < 1e-12
    assert factor == (0.1 * math.log(scaling['factor']) + 1 if scaling['rope_type'] == 'yarn' else 1.0)


@pytest.mark.parametrize('scaling,length', SCALINGS)
def test_tables_agree_with_transformers(scaling, length):
    from transformers import Qwen2Config
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    theta, hd = 1e6, 128
    c = Qwen2Config(hidden_size=8 * hd, num_attention_heads=8, max_position_embeddings=32768,
                    rope_parameters=dict(scaling, rope_theta=theta))
    if 'original_max_position_embeddings' in scaling:
        c.max_position_embeddings = scaling['original_max_position_embeddings']
    want, factor = ROPE_INIT_FUNCTIONS[scaling['rope_type']](c, torch.device('cpu'), seq_len=length)
    inv, got = rotary_frequencies(hd, theta, scaling, length)
    # theirs is computed in 32 bits: a power of up to 20 bits' exponent carries a few 2^-24 of its logarithm
    assert float(((inv - want.double()) / inv).abs().max()) < 64 * 2.0 ** -24
    assert abs(got - factor) < 1e-6


def test_default_and_explicit_factors():
    inv, factor = rotary_frequencies(64, 1e4)
    assert factor == 1.0 and float(inv[0]) == 1.0 and abs(float(inv[-1]) - 1e4 ** (-62 / 64)) < 1e-18
    assert rotary_frequencies(64, 1e4, {'rope_type': 'default'})[1] == 1.0
    y = {'rope_type': 'yarn', 'factor': 4.0, 'original_max_position_embeddings': 4096}
    assert rotary_frequencies(64, 1e4, dict(y, attention_factor=1.5))[1] == 1.5
    assert abs(rotary_frequencies(64, 1e4, dict(y, mscale=0.707, mscale_all_dim=1.0))[1]
               - (0.0707 * math.log(4) + 1) / (0.1 * math.log(4) + 1)) < 1e-15


def test_bad_tables_are_refused():
    for args in [(63, 1e4), (0, 1e4), (64, 1e4, {'rope_type': 'longrope', 'factor': 2.0}), (64, 1e4, {'rope_type': 'yarn', 'factor': 4.0}),
                 (64, 1e4, {'rope_type': 'linear', 'factor': 0.5}), (2, 1e4, {'rope_type': 'dynamic', 'factor': 2.0,
                                                                             'original_max_position_embeddings': 64})]:
        with pytest.raises(ValueError):
            rotary_frequencies(*args)
