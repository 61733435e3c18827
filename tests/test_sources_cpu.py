"""What the sources, scripts and build files may not hold: GPU code that writes through the scalar data cache (scalar stores, scalar
atomics, that cache's write-back and discard).  Kernels write memory with vector stores; comments and tools name no such instruction either."""
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TREES = ('neoradium_amd', 'include', 'oracle', 'tests', 'tools')
SUFFIXES = ('.hip', '.h', '.hpp', '.c', '.cc', '.cpp', '.cu', '.s', '.S', '.asm', '.ll', '.py', '.sh', '.mk', '.cmake', '.toml', '.cfg')
NAMES = ('Makefile', 'CMakeLists.txt')
SCALAR_WRITE = re.compile(r'(?:\b|_)s_(?:(?:buffer_|scratch_)?(?:store|atomic)(?:_|\b)|dcache_(?:wb|discard))', re.I)


def source_files():
    paths = [os.path.join(ROOT, f) for f in os.listdir(ROOT)]
    for tree in TREES:
        for folder, _, files in os.walk(os.path.join(ROOT, tree)):
            paths += [os.path.join(folder, f) for f in files]
    return sorted(p for p in paths if os.path.isfile(p) and (p.endswith(SUFFIXES) or os.path.basename(p) in NAMES))


@pytest.mark.parametrize('memory', ['', 'buffer_', 'scratch_'])
@pytest.mark.parametrize('op', ['store', 'atomic'])
def test_the_pattern_finds_scalar_writes(memory, op):
    assert SCALAR_WRITE.search(f'asm volatile("s_{memory}{op}_dwordx2 %0, %1, 0"')
    assert SCALAR_WRITE.search(f"op.startswith('s_{memory}{op}')")
    assert not SCALAR_WRITE.search(f'global_{op}_dwordx2 v[0:1], v[2:3], off')
    assert not SCALAR_WRITE.search(f'buffer_{op}_dwordx2 v[0:1], v2, s[0:3], 0')


@pytest.mark.parametrize('op', ['wb', 'wb_vol', 'discard', 'discard_x2'])
def test_the_pattern_finds_scalar_cache_writes(op):
    assert SCALAR_WRITE.search(f's_dcache_{op}')
    assert SCALAR_WRITE.search(f'__builtin_amdgcn_s_dcache_{op}()')


@pytest.mark.parametrize('text', ['s_load_dwordx2 s[0:1], s[2:3], 0x0', 's_buffer_load_dword s0, s[4:7], 0x0', 's_waitcnt lgkmcnt(0)'])
def test_the_pattern_leaves_scalar_reads(text):
    assert not SCALAR_WRITE.search(text)


def test_no_source_writes_through_the_scalar_cache():
    files = source_files()
    assert any(f.endswith('nrx_ldpc_dec3.hip') for f in files) and any(f.endswith('build.py') for f in files)
    found = []
    for path in files:
        with open(path, encoding='utf-8', errors='replace') as f:
            found += [f'{os.path.relpath(path, ROOT)}:{n}' for n, line in enumerate(f, 1) if SCALAR_WRITE.search(line)]
    assert not found, 'scalar stores, scalar atomics or scalar cache write-back named in: ' + ', '.join(found)
