"""Builds libvcgan_hip.so (hand-written HIP for gfx950) in-tree with hipcc.

No torch.utils.cpp_extension (it would hipify); plain `hipcc -c` per translation unit (in parallel) and one
`hipcc -shared` link.  Objects live in csrc/build/ (git-ignored), the library next to the sources.
"""
import os
import subprocess
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, 'csrc')
OBJ = os.path.join(CSRC, 'build')
LIB = os.path.join(CSRC, 'libvcgan_hip.so')
SOURCES = ['vc_testing.hip', 'vc_conv_igemm.hip', 'vc_conv_bf16.hip', 'vc_conv_wgrad.hip', 'vc_conv_small.hip', 'vc_conv_glu.hip', 'vc_conv_wino.hip', 'vc_elementwise.hip', 'vc_tables.hip', 'vc_ops.hip', 'vc_net.hip', 'vc_step.hip', 'vc_comm.hip',
           'vc_seq_norm.hip', 'vc_seq_conv.hip', 'vc_seq_scan.hip', 'vc_seq_scan_bwd.hip']
HEADERS = ['vc_internal.h', 'vc_host.h', 'vc_device_util.h', 'vc_wino.h', 'vc_tuned_igemm.h', 'vc_tuned_wgrad.h', 'vc_tuned_bf16.h', 'vc_seq.h', 'vc_seq_scan.h', os.path.join('..', '..', 'include', 'vc_cyclegan.h'),
           os.path.join('..', '..', 'include', 'vc_cyclegan_testing.h')]
# -packed-fp32-ops: no v_pk_{mul,add,fma}_f32 in any kernel.  Round 6: inside the bf16 train step, with the generator's filter-gradient GEMMs on
# their own stream, norm_bwd_v4_kernel now and then gave ONE 16-lane group (lanes 48-63 of one wave) wrong row sums from register contents that
# were bitwise the same as in a good launch (round-6 probe, in the git history: values as loaded identical, s1 / s2 different); 31 of 80 trials with the
# packed instructions, 0 of 240 without them in this translation unit or anywhere, at the same ms per step in every benched configuration
# (profiles/r06_wrong_lane_group.txt).  The cause is not established beyond that correlation; the instructions buy nothing here (every kernel
# that uses them is bound by memory or by MFMA), so the whole library is built without them.
FLAGS = ['--offload-arch=gfx950', '-O3', '-std=c++20', '-munsafe-fp-atomics', '-fPIC',
         '-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops',
         '-Wall', '-Wextra', '-Wno-unused-parameter']
HOST_NOISE = "is not a recognized feature for this target (ignoring feature)"    # the host half of each compile sees the device-only feature flag


def _run(cmd, cwd):
    r = subprocess.run(cmd, cwd=cwd, stderr=subprocess.PIPE, text=True)
    err = ''.join(l for l in r.stderr.splitlines(True) if HOST_NOISE not in l)
    if err:
        print(err, end='', flush=True)
    if r.returncode:
        raise subprocess.CalledProcessError(r.returncode, cmd)


def build_id(extra=()):
    """SHA-256 (first 16 hex digits) over every source and header the library is built from and the compiler flags.  The
    library carries the value it was built with (vc_build_id()); _lib.py recomputes it at import and refuses to load on
    a mismatch, so a library older or newer than the sources next to it can neither be tested nor benched (
    freshness was judged by mtime only, and the prebuilt .so travels to the GPU box next to sources with fresh mtimes)."""
    import hashlib
    h = hashlib.sha256()
    for f in sorted(SOURCES + HEADERS):
        h.update(os.path.basename(f).encode() + b'\0')
        with open(os.path.join(CSRC, f), 'rb') as fh:
            h.update(fh.read())
        h.update(b'\0')
    h.update(' '.join(FLAGS + list(extra) + os.environ.get('VC_EXTRA_FLAGS_ONLY', '').split()).encode())
    return h.hexdigest()[:16]


def _mtime(p):
    return os.path.getmtime(p) if os.path.exists(p) else 0.0


def _stale(target, deps):
    t = _mtime(target)
    return t == 0.0 or any(_mtime(d) > t for d in deps)


ID_FILE = LIB + '.buildid'


def needs_build():
    """True when the library is missing or was built from other sources / flags than the ones in the tree (content hash, not mtime)."""
    if not os.path.exists(LIB) or not os.path.exists(ID_FILE):
        return True
    return open(ID_FILE).read().strip() != build_id(os.environ.get('VC_EXTRA_FLAGS', '').split())


# ---- the torch binding of the sequence operators (host code; everything it calls of the library it gets by address at import)
BINDING_SOURCE = os.path.join(CSRC, 'vc_seq_torch.cpp')
BINDING = os.path.join(HERE, '_seq.so')
BINDING_FLAGS = ['-O2', '-std=c++17', '-fPIC', '-shared', '-Wall']


def binding_id():
    """Content hash of the binding's source, the header it is written against, its flags and the torch and Python it is built for."""
    import hashlib
    import sys
    import torch
    h = hashlib.sha256()
    for f in (BINDING_SOURCE, os.path.join(HERE, '..', 'include', 'vc_cyclegan.h')):
        with open(f, 'rb') as fh:
            h.update(fh.read())
        h.update(b'\0')
    h.update(' '.join(BINDING_FLAGS + [torch.__version__, sys.version]).encode())
    return h.hexdigest()[:16]


def binding_lacks():
    """What the binding cannot be built without and this machine has not got (None: nothing).  The C-ABI library needs none of it."""
    import shutil
    import sysconfig
    try:
        import torch
    except ImportError as e:
        return 'torch cannot be imported (%s)' % e
    cxx = os.environ.get('CXX', 'g++')
    if not shutil.which(cxx):
        return 'there is no host compiler %s' % cxx
    for header in (os.path.join(os.path.dirname(torch.__file__), 'include', 'torch', 'csrc', 'utils', 'pybind.h'), os.path.join(sysconfig.get_paths()['include'], 'Python.h')):
        if not os.path.exists(header):
            return 'there is no %s' % header
    return None


def build_binding(force=False, verbose=True):
    import sysconfig
    import torch
    bid, stamp = binding_id(), BINDING + '.buildid'
    if not force and os.path.exists(BINDING) and os.path.exists(stamp) and open(stamp).read().strip() == bid:
        return BINDING
    root = os.path.dirname(torch.__file__)
    cmd = [os.environ.get('CXX', 'g++')] + BINDING_FLAGS + ['-I' + os.path.join(root, 'include'), '-I' + os.path.join(root, 'include', 'torch', 'csrc', 'api', 'include'),
           '-I' + sysconfig.get_paths()['include'], '-DVC_BINDING_ID="%s"' % bid, BINDING_SOURCE, '-o', BINDING, '-L' + os.path.join(root, 'lib'),
           '-lc10', '-ltorch_cpu', '-ltorch', '-ltorch_python']
    if verbose:
        print('[vcgan] ' + ' '.join(cmd), flush=True)
    _run(cmd, CSRC)
    with open(stamp, 'w') as fh:
        fh.write(bid + '\n')
    return BINDING


def build(force=False, verbose=True):
    """The library, then the binding where it can be built; without it sequence.py says so at import, and everything else works."""
    lib = build_library(force, verbose)
    lacks = binding_lacks()
    if lacks is None:
        build_binding(force, verbose)
    else:
        print('[vcgan] the torch binding of the sequence operators is not built: ' + lacks, flush=True)
    return lib


def build_library(force=False, verbose=True):
    if not force and not needs_build():
        return LIB
    hipcc = os.environ.get('HIPCC', '/opt/rocm/bin/hipcc')
    os.makedirs(OBJ, exist_ok=True)
    hdrs = [os.path.join(CSRC, h) for h in HEADERS]
    extra = os.environ.get('VC_EXTRA_FLAGS', '').split()
    only = os.environ.get('VC_EXTRA_FLAGS_ONLY', '').split()      # experiments: the extra flags go to these translation units only
    bid = build_id(extra)

    def compile_one(src):
        obj = os.path.join(OBJ, src.replace('.hip', '.o'))
        stamp = src == 'vc_tables.hip'              # the translation unit that carries the build id: recompiled on every change of it
        if force or extra or stamp or _stale(obj, [os.path.join(CSRC, src)] + hdrs):
            cmd = [hipcc] + FLAGS + (extra if not only or src in only else []) + (['-DVC_BUILD_ID="%s"' % bid] if stamp else []) + ['-c', os.path.join(CSRC, src), '-o', obj]
            if verbose:
                print('[vcgan] ' + ' '.join(cmd), flush=True)
            _run(cmd, CSRC)
        return obj

    with ThreadPoolExecutor(max_workers=min(len(SOURCES), os.cpu_count() or 1)) as ex:
        objs = list(ex.map(compile_one, SOURCES))
    cmd = [hipcc, '--offload-arch=gfx950', '-shared', '-fPIC', '-o', LIB] + objs + ['-ldl']
    if verbose:
        print('[vcgan] ' + ' '.join(cmd), flush=True)
    subprocess.check_call(cmd, cwd=CSRC)
    with open(ID_FILE, 'w') as fh:
        fh.write(bid + '\n')
    return LIB


if __name__ == '__main__':
    build(force=True)
