"""Build libseedplane_hip.so in-tree with hipcc for gfx950.

    python -m seedplane_amd.build            # the library
    python -m seedplane_amd.build sanitized  # a host-sanitized copy for CPU tests (_build/, not shipped)
"""
import os
import subprocess
import sys
import tempfile
from pathlib import Path

PKG = Path(__file__).resolve().parent
SOURCES = [PKG / 'csrc' / 'sp_engine.hip', PKG / 'csrc' / 'sp_paged.hip']
OUT = PKG / 'libseedplane_hip.so'
HIPCC = os.environ.get('HIPCC', '/opt/rocm/bin/hipcc')

FLAGS = ['--offload-arch=gfx950', '-O3', '-std=c++17', '-fPIC',
         # packed fp32 instructions stay off (hipcc -O3 would otherwise form v_pk_* fp32 ops)
         '-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops',
         '-Wno-pass-failed']


def _errors(text):
    return '\n'.join(l for l in (text or '').splitlines() if 'is not a recognized feature for this target' not in l)


def _compile(flags, out):
    """Every source to an object of its own (in parallel), then one shared library; returns the compilers' messages."""
    with tempfile.TemporaryDirectory() as d:
        objects = [str(Path(d) / (src.stem + '.o')) for src in SOURCES]
        jobs = [subprocess.Popen([HIPCC, *flags, '-c', '-o', obj, str(src)], stdout=subprocess.DEVNULL, stderr=subprocess.PIPE,
                                 text=True) for src, obj in zip(SOURCES, objects)]
        texts = [_errors(j.communicate()[1]) for j in jobs]
        for j, text, src in zip(jobs, texts, SOURCES):
            if j.returncode != 0:
                raise RuntimeError(f'hipcc failed ({j.returncode}) on {src.name}:\n{text}')
        tmp = out.with_suffix('.so.tmp')
        r = subprocess.run([HIPCC, *flags, '-shared', '-o', str(tmp), *objects], capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f'hipcc failed ({r.returncode}):\n{_errors(r.stderr)}')
        os.replace(tmp, out)
    return '\n'.join(t for t in texts if t.strip())


def build(verbose=False):
    text = _compile(FLAGS, OUT)
    if verbose and text:
        print(text, file=sys.stderr)
    return OUT


# Host code only under AddressSanitizer + UndefinedBehaviorSanitizer (-Xarch_host before each -fsanitize=; the gfx950
# code is built as usual).  CPU tests load it through SEEDPLANE_HIP_LIB with the clang ASan runtime preloaded.
SAN_OUT = PKG.parent / '_build' / 'libseedplane_hip_san.so'
SAN_FLAGS = ['--offload-arch=gfx950', '-O1', '-std=c++17', '-fPIC',
             '-Xarch_host', '-g', '-Xarch_host', '-fno-omit-frame-pointer',
             '-Xarch_host', '-fsanitize=address', '-Xarch_host', '-fsanitize=undefined',
             '-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops', '-Wno-pass-failed']


def asan_runtime():
    """The clang AddressSanitizer runtime that matches hipcc's compiler."""
    found = sorted(Path('/opt/rocm/lib/llvm/lib/clang').glob('*/lib/linux/libclang_rt.asan-x86_64.so'))
    if not found:
        raise FileNotFoundError('clang ASan runtime not found under /opt/rocm/lib/llvm/lib/clang')
    return found[-1]


def build_sanitized(out=SAN_OUT):
    out.parent.mkdir(parents=True, exist_ok=True)
    _compile(SAN_FLAGS, out)
    return out


if __name__ == '__main__':
    print(build_sanitized() if sys.argv[1:] == ['sanitized'] else build(verbose=True))
