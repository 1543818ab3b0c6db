"""Build libnerf_amd.so (gfx950) in-tree with hipcc, and the host module that reads tensor lists (`_tensor_lists`).

    python -m nerf_amd.build [--force]

Each .hip translation unit is compiled to an object with its own flags, then linked into
`nerf_amd/lib/libnerf_amd.so`.  hipcc cross-compiles for gfx950 without a GPU present.
"""
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, 'csrc')
LIBDIR = os.path.join(HERE, 'lib')
OBJDIR = os.path.join(LIBDIR, 'obj')
LIB = os.path.join(LIBDIR, 'libnerf_amd.so')

# (no packed fp32 instructions, which the compiler forms from ordinary float code by itself: a precaution, every kernel is
# written and tested as scalar fp32 arithmetic.  They gain nothing here: the training step takes 46.5 ms with and without)
COMMON = ['--offload-arch=gfx950', '-O3', '-fPIC', '-std=c++17', '-Wall', '-Wno-unused-function',
          '-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops']
# translation unit -> extra flags.  The sampling / compositing kernels must round every fp32
# operation separately (parity with the reference's op-by-op torch arithmetic).
# mlp_bf16.hip is compiled in parts (-DNERF_NET_PART=p): the chain kernels of each large network geometry take
# minutes to compile, so each gets its own object and they build side by side.
UNITS = {
    'api.o': ('api.hip', []),
    'sampling.o': ('sampling.hip', ['-ffp-contract=off']),
    'composite.o': ('composite.hip', ['-ffp-contract=off']),
    'sar_pulse.o': ('sar_pulse.hip', []),
    'gemm_f32.o': ('gemm_f32.hip', []),
    'optimizer.o': ('optimizer.hip', []),
    # VGPR-form matrix-core instructions where an accumulator tile lives in the vector registers: the outputs of the
    # larger launches exceed the 256 accumulation registers, and the default form copies such tiles in and out
    # of them around every product (layer 4's launch: 1.10 -> 0.86 ms)
    'wgrad8.o': ('wgrad8.hip', ['-mllvm', '-amdgpu-mfma-vgpr-form']),
}
UNITS.update({'mlp_bf16_p%d.o' % p: ('mlp_bf16.hip', ['-DNERF_NET_PART=%d' % p]) for p in range(8)})   # default contraction
LISTS_SRC = os.path.join(CSRC, 'tensor_lists.cpp')
LISTS = os.path.join(HERE, '_tensor_lists.so')
LISTS_RECORD = os.path.join(OBJDIR, 'tensor_lists.txt')         # what LISTS was built with
JOBS = int(os.environ.get('MAX_JOBS', '8'))


def _hipcc():
    for c in ('/opt/rocm/bin/hipcc', 'hipcc'):
        if os.path.isabs(c) and os.path.exists(c):
            return c
    return 'hipcc'


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _lists_command():
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths
    libdir = os.path.join(os.path.dirname(torch.__file__), 'lib')
    return (['g++', '-O2', '-std=c++17', '-fPIC', '-shared', '-Wall',
             '-D_GLIBCXX_USE_CXX11_ABI=%d' % torch.compiled_with_cxx11_abi()]
            + ['-I' + d for d in include_paths() + [sysconfig.get_paths()['include']]]
            + [LISTS_SRC, '-o', LISTS, '-L' + libdir, '-ltorch_python', '-ltorch_cpu', '-lc10'])


def lists_record():
    """The host module goes by torch's C++ headers and by Python's: its command and both versions."""
    import torch
    return '\n'.join([' '.join(_lists_command()), torch.__version__, sys.version])


def lists_stale():
    if _stale(LISTS, [LISTS_SRC, os.path.abspath(__file__)]) or not os.path.exists(LISTS_RECORD):
        return True
    with open(LISTS_RECORD) as f:
        return f.read() != lists_record()


def build(force=False, verbose=True):
    os.makedirs(OBJDIR, exist_ok=True)
    headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(('.h', '.inc'))]
    headers.append(os.path.join(os.path.dirname(HERE), 'include', 'nerf_amd.h'))
    headers.append(os.path.abspath(__file__))
    jobs, objs = [], []
    for name, (unit, extra) in UNITS.items():
        src = os.path.join(CSRC, unit)
        obj = os.path.join(OBJDIR, name)
        objs.append(obj)
        if force or _stale(obj, [src] + headers):
            jobs.append([_hipcc()] + COMMON + extra + ['-c', src, '-o', obj])
    host = [_lists_command()] if force or lists_stale() else []
    for f in os.listdir(OBJDIR):                      # objects of an older unit list must not be linked
        if f.endswith('.o') and f not in UNITS:
            os.remove(os.path.join(OBJDIR, f))

    def run(cmd):
        if verbose:
            print(' '.join(cmd), flush=True)
        subprocess.run(cmd, check=True)

    with ThreadPoolExecutor(max_workers=min(JOBS, max(1, len(jobs + host)))) as ex:
        list(ex.map(run, jobs + host))
    if host:
        with open(LISTS_RECORD, 'w') as f:
            f.write(lists_record())
    if jobs or force or _stale(LIB, objs):
        run([_hipcc(), '--offload-arch=gfx950', '-shared', '-fPIC', '-o', LIB] + objs)
    return LIB


if __name__ == '__main__':
    print(build(force='--force' in sys.argv))
