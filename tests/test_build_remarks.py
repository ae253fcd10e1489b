"""The build reads how much scratch memory each kernel takes, whatever its compilers print at the same time."""
import os
import stat

import pytest

from qmoe_amd import build

REMARK = '{0}.hip:7:1: remark: Function Name: {1} [-Rpass-analysis=kernel-resource-usage]\n' \
         '    7 | __global__ void {1}(int *p) {{\n      | ^\n' \
         '{0}.hip:7:1: remark:     VGPRs: 40 [-Rpass-analysis=kernel-resource-usage]\n' \
         '{0}.hip:7:1: remark:     ScratchSize [bytes/lane]: {2} [-Rpass-analysis=kernel-resource-usage]\n'

# Prints what a compiler of all its sources side by side would: the sources' remarks character by character in turn.
COMPILER = '''#!/usr/bin/env python3
import os, sys
if len(sys.argv) > 2 and '-o' in sys.argv:
    open(sys.argv[sys.argv.index('-o') + 1], 'w').write('built')
texts = [open(a).read() for a in sys.argv[1:] if a.endswith('.hip')]
for i in range(max(map(len, texts), default=0)):
    for text in texts:
        os.write(1, text[i:i + 1].encode())
'''


def build_of(tmp_path, monkeypatch, sizes):
    """build_library of a source for each of sizes, whose kernels take so much scratch memory"""
    compiler = tmp_path / 'compiler'
    compiler.write_text(COMPILER)
    compiler.chmod(compiler.stat().st_mode | stat.S_IXUSR)
    sources = []
    for name, of in sizes.items():
        source = tmp_path / (name + '.hip')
        source.write_text(''.join(REMARK.format(name, '%s_%d' % (name, i), size) for i, size in enumerate(of)))
        sources.append(str(source))
    monkeypatch.setenv('HIPCC', str(compiler))
    monkeypatch.setattr(build, 'SOURCES', sources)
    monkeypatch.setattr(build, 'LIB_PATH', str(tmp_path / 'library.so'))
    monkeypatch.setattr(build, 'build_tensor_args', lambda: None)
    monkeypatch.setattr(build, 'SPILLS_ACCEPTED', {'one_1': 36})
    return build.build_library()


def test_what_spills_is_found_in_every_source(tmp_path, monkeypatch):
    sizes = {'one': [0, 36, 0], 'three': [0] * 5, 'seventeen': [0, 0, 0]}
    assert os.path.exists(build_of(tmp_path, monkeypatch, sizes))
    for name, at in (('one', 2), ('three', 4), ('seventeen', 0)):
        more = {k: list(v) for k, v in sizes.items()}
        more[name][at] = 12
        with pytest.raises(RuntimeError, match="^kernels that spill registers to scratch memory: {'%s_%d': 12}$" % (name, at)):
            build_of(tmp_path, monkeypatch, more)
        assert not os.path.exists(build.LIB_PATH)       # nor one of other sources


def test_a_source_of_whose_kernels_nothing_is_said(tmp_path, monkeypatch):
    with pytest.raises(RuntimeError, match='nothing about the kernels'):
        build_of(tmp_path, monkeypatch, {'one': [0, 0], 'two': []})


def test_remarks():
    text = ''.join(REMARK.format('a', 'k%d' % i, size) for i, size in enumerate((0, 8, 0, 4)))
    assert build.kernels_with_scratch(text) == {'k1': 8, 'k3': 4} and build.kernels_with_scratch('') == {}
    lines = text.splitlines(keepends=True)
    for lost in range(len(lines)):          # a line of a name or a size lost, or cut in two
        if 'Function Name' in lines[lost] or 'ScratchSize' in lines[lost]:
            cut = lines[lost].index('k') + 1 if 'Function Name' in lines[lost] else lines[lost].index('lane') + 2
            for instead in ('', lines[lost][:cut] + '\n' + lines[lost][cut:]):
                with pytest.raises(RuntimeError):
                    build.kernels_with_scratch(''.join(lines[:lost]) + instead + ''.join(lines[lost + 1:]))
    pair = text[:60], REMARK.format('b', 'other', 0)
    mixed = ''.join(x + y for x, y in zip(*pair)) + text[60:]
    with pytest.raises(RuntimeError):
        build.kernels_with_scratch(mixed)
