"""The decay-attention argument blocks have one layout in the C header, in ctypes and in the packed form that calls use."""
import os
import shutil
import subprocess

import pytest

from bdm_b200 import _lib, decay

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'include', 'bdm_b200.h')
BLOCKS = [('bdm_decay_walk_args', _lib.DecayWalkArgs, decay._WALK), ('bdm_decay_step_args', _lib.DecayStepArgs, decay._STEP)]


@pytest.mark.parametrize('name,block,packed', BLOCKS)
def test_packed_blocks_match_ctypes(name, block, packed):
    import ctypes
    assert packed.size == ctypes.sizeof(block)
    values, want = [], {}
    for field, kind in block._fields_:
        n = getattr(kind, '_length_', 1)
        got = [len(values) + 1 + i for i in range(n)]
        values += got
        want[field] = got if n > 1 else got[0]
    a = block.from_buffer_copy(packed.pack(*values))
    for field, value in want.items():
        x = getattr(a, field)
        assert (list(x) if isinstance(value, list) else x) == value, field


@pytest.mark.parametrize('name,block,packed', BLOCKS)
def test_ctypes_blocks_match_the_header(name, block, packed, tmp_path):
    import ctypes
    cc = shutil.which('gcc') or shutil.which('cc')
    if cc is None:
        pytest.skip('no C compiler')
    fields = [f for f, _ in block._fields_]
    source = tmp_path / 'layout.c'
    source.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "%s"\nint main(void) {\n printf("%%zu", sizeof(%s));\n%s return 0;\n}\n'
                      % (HEADER, name, ''.join(f' printf(" %zu", offsetof({name}, {f}));\n' for f in fields)))
    program = tmp_path / 'layout'
    subprocess.run([cc, '-o', str(program), str(source)], check=True)
    got = [int(x) for x in subprocess.run([str(program)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [ctypes.sizeof(block)] + [getattr(block, f).offset for f in fields]
