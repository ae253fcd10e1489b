"""Compiles libsub1_hip.so for gfx950 with hipcc (cross-compiles without a GPU), and
the Python extension that takes tensors apart for it with g++."""
import concurrent.futures
import os
import re
import subprocess
import sysconfig
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
LIB_PATH = os.path.join(HERE, 'libsub1_hip.so')
TENSOR_ARGS_PATH = os.path.join(HERE, '_tensor_args.so')
SOURCES = [os.path.join(HERE, 'csrc', 'sub1_kernels.hip'),
           os.path.join(HERE, 'csrc', 'sub1_pack.hip'),
           os.path.join(HERE, 'csrc', 'sub1_prepared.hip'),
           os.path.join(HERE, 'csrc', 'sub1_tiles.hip'),
           os.path.join(HERE, 'csrc', 'mx4_matrix.hip'),
           os.path.join(HERE, 'csrc', 'mx4_layer.hip'),
           os.path.join(HERE, 'csrc', 'mx8_matrix.hip'),
           os.path.join(HERE, 'csrc', 'norm.hip'),
           os.path.join(HERE, 'csrc', 'routing.hip'),
           os.path.join(HERE, 'csrc', 'sub1_tables.cpp')]

HIPCC_FLAGS = [
    '-O3', '--offload-arch=gfx950', '-fPIC', '-std=c++17',
    # keep the compiler from forming packed fp32 instructions
    '-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops',
    # registers and scratch memory per kernel, read back below
    '-Rpass-analysis=kernel-resource-usage',
    '-I' + os.path.join(ROOT, 'include'), '-I' + os.path.join(HERE, 'csrc'),
]


JOBS = 8      # compilers at a time: 95 to 110 s in place of 200


def kernels_with_scratch(compiler_output):
    """{kernel: bytes of scratch memory per lane} for the kernels that spill registers, from the
    compiler's resource-usage remarks on one source.  Raises RuntimeError where these are not a
    name and a size in turn (lines cut into each other, one of them lost)."""
    found, name, names, sizes = {}, None, 0, 0
    for line in compiler_output.splitlines():
        m = re.search(r'remark: Function Name: (\S+) \[-Rpass', line)
        if m:
            if name:
                raise RuntimeError('no scratch size of kernel %s in the compiler\'s remarks' % name)
            name, names = m.group(1), names + 1
        m = re.search(r'remark:\s+ScratchSize \[bytes/lane\]: (\d+) \[-Rpass', line)
        if m:
            if not name:
                raise RuntimeError('a scratch size of no kernel in the compiler\'s remarks')
            if int(m.group(1)):
                found[name] = int(m.group(1))
            name, sizes = None, sizes + 1
    if not names == sizes == compiler_output.count('Function Name') == compiler_output.count('ScratchSize'):
        raise RuntimeError('the compiler\'s remarks cannot be read: %d names and %d scratch sizes of %d and %d' % (
            names, sizes, compiler_output.count('Function Name'), compiler_output.count('ScratchSize')))
    return found


# Kernels known to spill, and how many bytes per lane: the fused kernel's form for
# tokens grouped by expert keeps four tokens' sums per lane.
SPILLS_ACCEPTED = {'_ZN12_GLOBAL__N_125moe_prepared_fused_kernelILb1ELb0ELb0EEEvNS_12PreparedArgsE': 36}


def torch_mark():
    """What the extension says of the torch that it was built against, of the one installed."""
    import torch
    return 'qmoe_amd, built against torch ' + torch.__version__


def build_tensor_args():
    """Builds the extension module against the installed torch's headers."""
    import torch
    from torch.utils import cpp_extension
    cmd = [os.environ.get('CXX', 'g++'), '-O2', '-fPIC', '-shared', '-std=c++17', '-fvisibility=hidden',
           '-D_GLIBCXX_USE_CXX11_ABI=%d' % torch._C._GLIBCXX_USE_CXX11_ABI,
           '-DSUB1_TORCH_VERSION="%s"' % torch.__version__,
           '-I' + os.path.join(ROOT, 'include'), os.path.join(HERE, 'csrc', 'tensor_args.cpp')]
    cmd += ['-isystem' + path for path in cpp_extension.include_paths() + [sysconfig.get_paths()['include']]]
    cmd += ['-L' + path for path in cpp_extension.library_paths()]
    cmd += ['-ltorch_python', '-ltorch_cpu', '-lc10', '-o', TENSOR_ARGS_PATH]
    res = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if res.returncode != 0:
        raise RuntimeError('g++ failed:\n' + res.stdout)
    return TENSOR_ARGS_PATH


def build_library(verbose=False):
    """Builds the library and the extension; refuses a build in which a kernel spills registers
    to scratch memory beyond what SPILLS_ACCEPTED lists.  The kernels are
    written to fit their registers (72 to 96 of the 128 that 16 wavefronts per
    compute unit leave a lane), and a spill in a walk costs more than any of
    the tunings measured; one build of the one-token launch that spilled 12
    registers also gave results that differed from run to run (cause not
    established; the code was restructured to fit)."""
    build_tensor_args()
    hipcc = os.environ.get('HIPCC', '/opt/rocm/bin/hipcc')

    def run(cmd):
        res = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
        if res.returncode != 0:
            raise RuntimeError('hipcc failed:\n' + res.stdout)
        return res.stdout

    # A compiler each, whose output is read by itself: several that write to one pipe cut each other's lines.
    with tempfile.TemporaryDirectory() as objects, concurrent.futures.ThreadPoolExecutor(JOBS) as jobs:
        into = [os.path.join(objects, os.path.basename(source) + '.o') for source in SOURCES]
        outputs = list(jobs.map(lambda source, o: run([hipcc] + HIPCC_FLAGS + ['-c', source, '-o', o]), SOURCES, into))
        spilling = {}
        for source, output in zip(SOURCES, outputs):
            if source.endswith('.hip') and 'Function Name' not in output:
                raise RuntimeError('the compiler says nothing about the kernels of ' + source)
            spilling.update((k, v) for k, v in kernels_with_scratch(output).items() if v > SPILLS_ACCEPTED.get(k, 0))
        if spilling:
            if os.path.exists(LIB_PATH):      # what is there is of other sources
                os.remove(LIB_PATH)
            raise RuntimeError('kernels that spill registers to scratch memory: %s' % spilling)
        run([hipcc, '--offload-arch=gfx950', '-fPIC', '-shared'] + into + ['-o', LIB_PATH])
    if verbose:
        print('\n'.join(l for l in ''.join(outputs).splitlines() if 'kernel-resource-usage' not in l
                        and not l.lstrip().startswith(('|', '^')) and '__global__' not in l))
    return LIB_PATH


def tensor_args_fit():
    """Whether the extension is there and of the installed torch (looked up in the file: a
    module that has been loaded cannot be loaded again once it is rebuilt)."""
    try:
        with open(TENSOR_ARGS_PATH, 'rb') as f:
            return torch_mark().encode() + b'\0' in f.read()
    except FileNotFoundError:
        return False


def build_what_is_missing():
    """For programs that use what is built: builds only what is not there."""
    if not os.path.exists(LIB_PATH):
        build_library()
    elif not tensor_args_fit():
        build_tensor_args()


if __name__ == '__main__':
    print(build_library(verbose=True))
