"""The paged operators' host code (argument checks, the attention plan) under AddressSanitizer and UndefinedBehaviorSanitizer, as
tests/test_host_sanitizer.py runs the rest."""
import os
import subprocess
import sys

import pytest

from seedplane_amd import build as B
from test_host_sanitizer import ROOT, _sanitized_lib


def test_paged_host_code_is_clean_under_asan_and_ubsan():
    try:
        rt = B.asan_runtime()
    except FileNotFoundError as e:
        pytest.skip(str(e))
    env = dict(os.environ, LD_PRELOAD=str(rt), SEEDPLANE_HIP_LIB=str(_sanitized_lib()),
               ASAN_OPTIONS='detect_leaks=0:halt_on_error=1:abort_on_error=1', UBSAN_OPTIONS='halt_on_error=1:print_stacktrace=1')
    r = subprocess.run([sys.executable, '-m', 'pytest', '-q', '-p', 'no:cacheprovider', '-m', 'not gpu',
                        str(ROOT / 'tests' / 'test_paged_plan.py'), str(ROOT / 'tests' / 'test_paged_refusals.py')],
                       cwd=str(ROOT), env=env, capture_output=True, text=True, timeout=900)
    tail = (r.stdout or '')[-3000:] + (r.stderr or '')[-3000:]
    assert r.returncode == 0, tail
    assert 'ERROR: AddressSanitizer' not in tail and 'runtime error' not in tail, tail
    assert ' passed' in r.stdout
