"""Build the HIP library in-tree:  python -m ga_gan_amd.build  (hipcc, gfx950 only).

Every csrc/*.hip is compiled to an object of its own (in parallel) and the objects are linked into
libsgops.so; csrc/sg_torch.cpp (host code: the operators' PyTorch side) is compiled into _sg_torch.so.  Staleness is
decided by content, not by time stamps: each object carries a stamp with the digest of its source, of every header and of
the compiler flags, the way the reference keys its plugin build directory by a digest of the op's sources
(torch_utils/custom_ops.py:88-104).  The whole build runs under an
exclusive file lock, so that several ranks importing a stale tree at once build it once and the others wait
(the reference's FileBaton, torch_utils/custom_ops.py:105-115).
"""
import concurrent.futures
import fcntl
import glob
import hashlib
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
OUT = os.path.join(HERE, 'libsgops.so')
TORCH_OUT = os.path.join(HERE, '_sg_torch.so')
TORCH_SRC = os.path.join(HERE, 'csrc', 'sg_torch.cpp')
OBJ_DIR = os.path.join(HERE, 'build')
# Without packed float32 arithmetic: the compiler forms v_pk_{add,mul,fma}_f32 from ordinary scalar code, and some of their operand
# forms have given wrong results on MI355X now and then.  (The host pass warns that it does not know the feature.)
CFLAGS = ['-O3', '-std=c++17', '--offload-arch=gfx950', '-fPIC', '-Wall', '-Wno-unused-function',
          '-Wno-unused-const-variable', '-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops']
# per-source additions: in the band and one-pass up-sampling kernels the vectoriser's pairs of adjacent scalars only cost moves.
EXTRA_CFLAGS = {'sg_band3x3': ['-fno-slp-vectorize'], 'sg_convup_fir': ['-fno-slp-vectorize']}


def sources():
    return sorted(glob.glob(os.path.join(HERE, 'csrc', '*.hip')))


def headers():
    return sorted(glob.glob(os.path.join(HERE, 'csrc', '*.h')) + glob.glob(os.path.join(ROOT, 'include', '*.h')))


def _digest(paths, extra=''):
    h = hashlib.md5(extra.encode())
    for path in paths:
        h.update(os.path.basename(path).encode())
        with open(path, 'rb') as f:
            h.update(f.read())
    return h.hexdigest()


def _read(path):
    try:
        with open(path) as f:
            return f.read()
    except OSError:
        return None


def _plan():
    """[(source, object, stamp path, wanted digest)] and the digest the linked library must carry."""
    common = _digest(headers(), ' '.join(CFLAGS))
    items = []
    for src in sources():
        stem = os.path.splitext(os.path.basename(src))[0]
        items.append((src, os.path.join(OBJ_DIR, stem + '.o'), os.path.join(OBJ_DIR, stem + '.md5'),
                      _digest([src], common + ' '.join(EXTRA_CFLAGS.get(stem, [])))))
    return items, hashlib.md5(''.join(i[3] for i in items).encode()).hexdigest()


def _torch_plan():
    """(compiler command, wanted digest) of the PyTorch side."""
    import sysconfig
    import torch
    from torch.utils import cpp_extension
    lib = os.path.join(os.path.dirname(torch.__file__), 'lib')
    flags = ['-O2', '-std=c++17', '-fPIC', '-shared', '-Wall', '-Wno-unknown-pragmas', '-D__HIP_PLATFORM_AMD__=1', '-DUSE_ROCM=1',
             f'-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}']
    include = [os.path.join(ROOT, 'include'), *cpp_extension.include_paths(), '/opt/rocm/include', sysconfig.get_paths()['include']]
    # (torch's headers as system headers: their warnings are not this file's)
    cmd = [os.environ.get('CXX', 'g++'), *flags, *[a for d in include for a in (('-I' if d.startswith(ROOT) else '-isystem'), d)], TORCH_SRC,
           '-L', lib, '-ltorch', '-ltorch_cpu', '-ltorch_python', '-ltorch_hip', '-lc10', '-lc10_hip', '-ldl']
    return cmd, _digest([TORCH_SRC] + headers(), ' '.join(flags) + torch.__version__)


def is_stale():
    _, want = _plan()
    _, torch_want = _torch_plan()
    return (not os.path.isfile(OUT) or _read(os.path.join(OBJ_DIR, 'libsgops.md5')) != want
            or not os.path.isfile(TORCH_OUT) or _read(os.path.join(OBJ_DIR, '_sg_torch.md5')) != torch_want)


def build(force=False, verbose=True, jobs=None):
    if not force and not is_stale():
        return OUT
    os.makedirs(OBJ_DIR, exist_ok=True)
    with open(os.path.join(OBJ_DIR, '.lock'), 'w') as lock:
        fcntl.flock(lock, fcntl.LOCK_EX)              # one builder per tree; the others wait here ...
        try:
            if not force and not is_stale():          # ... and find the work done
                return OUT
            hipcc = os.environ.get('HIPCC', '/opt/rocm/bin/hipcc')
            include = ['-I', os.path.join(ROOT, 'include'), '-I', os.path.join(HERE, 'csrc')]
            items, want = _plan()
            todo = [i for i in items if force or not os.path.isfile(i[1]) or _read(i[2]) != i[3]]

            def compile_one(item):
                src, obj, stamp, digest = item
                stem = os.path.splitext(os.path.basename(src))[0]
                cmd = [hipcc, *CFLAGS, *EXTRA_CFLAGS.get(stem, []), *include, '-c', src, '-o', obj]
                if verbose:
                    print(' '.join(cmd), flush=True)
                subprocess.run(cmd, check=True)
                with open(stamp, 'w') as f:
                    f.write(digest)

            torch_cmd, torch_want = _torch_plan()
            torch_stamp = os.path.join(OBJ_DIR, '_sg_torch.md5')

            def compile_torch():
                if not force and os.path.isfile(TORCH_OUT) and _read(torch_stamp) == torch_want:
                    return
                tmp = TORCH_OUT + f'.tmp{os.getpid()}'
                cmd = [*torch_cmd, '-o', tmp]
                if verbose:
                    print(' '.join(cmd), flush=True)
                subprocess.run(cmd, check=True)
                os.replace(tmp, TORCH_OUT)
                with open(torch_stamp, 'w') as f:
                    f.write(torch_want)

            jobs = jobs or min(len(todo) + 1, int(os.environ.get('MAX_JOBS', 0)) or os.cpu_count() or 1, 16)
            with concurrent.futures.ThreadPoolExecutor(max_workers=jobs) as pool:
                glue = pool.submit(compile_torch)
                list(pool.map(compile_one, todo))
                glue.result()
            tmp = OUT + f'.tmp{os.getpid()}'
            cmd = [hipcc, '--offload-arch=gfx950', '-shared', '-fPIC', *[i[1] for i in items], '-o', tmp]
            if verbose:
                print(' '.join(cmd), flush=True)
            subprocess.run(cmd, check=True)
            os.replace(tmp, OUT)                      # a process that has the old library mapped keeps its copy
            with open(os.path.join(OBJ_DIR, 'libsgops.md5'), 'w') as f:
                f.write(want)
        finally:
            fcntl.flock(lock, fcntl.LOCK_UN)
    return OUT


if __name__ == '__main__':
    build(force='--force' in sys.argv)
