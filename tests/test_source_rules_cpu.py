"""What no committed source, script or record may hold: instructions that write through the scalar data cache (GPU code writes through vector stores)."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FOLDERS = ('include', 'oracle', 'perf', 'pixparse_amd', 'profiles', 'scripts', 'tests')
# scalar stores and atomics, and that cache's write-back and discard; put together from parts, so that this file does not name them
FORBIDDEN = re.compile(r'\bs_' + r'(?:(?:buffer_|scratch_)?(?:store|atomic)_|dcache_(?:wb|discard))|' + 'amdgcn_s_' + r'(?:dcache_wb|buffer_store)')


def test_the_pattern_finds_what_it_is_for():
    for name in ('store_dwordx2', 'dcache_wb', 'atomic_add', 'buffer_store_dword', 'scratch_store_dword', 'dcache_discard'):
        assert FORBIDDEN.search('\t' + 's_' + name + ' %0')
    assert not FORBIDDEN.search('buffer_store_dwordx4 s_load_dwordx2 global_atomic_add ds_store_b32 s_dcache_inv')


def test_nothing_writes_through_the_scalar_data_cache():
    found = []
    for folder in FOLDERS:
        for path, _, files in os.walk(os.path.join(ROOT, folder)):
            for f in files:
                if f.endswith(('.so', '.o', '.pyc', '.safetensors')):
                    continue
                with open(os.path.join(path, f), errors='replace') as fh:
                    found += [f'{os.path.join(path, f)}:{i}' for i, line in enumerate(fh, 1) if FORBIDDEN.search(line)]
    assert not found, found
