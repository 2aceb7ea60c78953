"""C and C++ programs that fill the header's descriptors from read-only data compile without a cast or a warning."""
import subprocess
from pathlib import Path

import pytest

INCLUDE = Path(__file__).resolve().parents[1] / 'include'
SOURCE = '''
#include "seedplane_hip.h"
static const float scales[4] = {1, 1, 1, 1};
static const double frequencies[32] = {0};
int describe(void *k, void *v, sp_paged_kv *kv, sp_rotary *rotary) {
    kv->k_dev = k; kv->v_dev = v;
    kv->k_scale_dev = scales; kv->v_scale_dev = &scales[2];
    kv->scale_block = 0;
    rotary->inv_freq_dev = frequencies;
    return kv->k_scale_dev == scales;
}
'''


@pytest.mark.parametrize('compiler,name', [(['gcc', '-std=c99'], 'a.c'), (['g++', '-std=c++17'], 'a.cpp')])
def test_descriptors_of_read_only_scales(tmp_path, compiler, name):
    (tmp_path / name).write_text(SOURCE)
    r = subprocess.run([*compiler, '-Wall', '-Wextra', '-Werror', '-fsyntax-only', '-I', str(INCLUDE), str(tmp_path / name)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
