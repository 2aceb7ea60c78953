"""The host code of caches in blocks, the page pool and the beam selection under AddressSanitizer and UndefinedBehaviorSanitizer, as
tests/test_paged_sanitizer.py runs the other paged operators."""
import os
import subprocess
import sys

import pytest

from seedplane_amd import build as B
from test_host_sanitizer import ROOT, _sanitized_lib


def test_host_code_is_clean_under_asan_and_ubsan():
    try:
        rt = B.asan_runtime()
    except FileNotFoundError as e:
        pytest.skip(str(e))
    env = dict(os.environ, LD_PRELOAD=str(rt), SEEDPLANE_HIP_LIB=str(_sanitized_lib()),
               ASAN_OPTIONS='detect_leaks=0:halt_on_error=1:abort_on_error=1', UBSAN_OPTIONS='halt_on_error=1:print_stacktrace=1')
    r = subprocess.run([sys.executable, '-m', 'pytest', '-q', '-p', 'no:cacheprovider', '-m', 'not gpu', '--deselect',
                        'tests/test_blocks_refusals.py::test_python_refusals', str(ROOT / 'tests' / 'test_blocks_refusals.py'),
                        str(ROOT / 'tests' / 'test_pages_refusals.py')],
                       cwd=str(ROOT), env=env, capture_output=True, text=True, timeout=900)
    tail = (r.stdout or '')[-3000:] + (r.stderr or '')[-3000:]
    assert r.returncode == 0, tail
    assert 'ERROR: AddressSanitizer' not in tail and 'runtime error' not in tail, tail
    assert ' passed' in r.stdout
