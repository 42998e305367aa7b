"""Wait states between a vector instruction that writes a scalar register and the memory
instruction that reads it.

On the GFX9 family a vector-memory instruction may not read a scalar register (its resource
or its scalar offset) in the five wait states after a vector instruction, v_readfirstlane above all,
wrote it.  The compiler keeps them for its own instructions; it does not look inside asm statements.
So the assembly of every kernel source with such a load in an asm statement is checked here as built."""
import concurrent.futures as cf
import os
import re
import subprocess

import pytest

from musc_hip import build

WAIT_STATES = 5
MEMORY = ('buffer_', 'global_', 'flat_', 'scratch_')


def _scalars(operand: str) -> set[str]:
    out = {f's{i}' for m in re.finditer(r'\bs\[(\d+):(\d+)\]', operand) for i in range(int(m[1]), int(m[2]) + 1)}
    return out | {m[0] for m in re.finditer(r'\bs\d+\b|\bvcc\b', operand)}


def _operands(ins: str) -> list[str]:
    parts = ins.split(None, 1)
    return [x.strip() for x in re.split(r',(?![^\[]*\])', parts[1])] if len(parts) > 1 else []


def _written(ins: str) -> set[str]:
    """Scalar registers that a vector instruction writes: lane reads and comparisons their first
    operand, carries and scaled divisions their second."""
    ops, name = _operands(ins), ins.split()[0]
    if name.startswith(('v_readfirstlane', 'v_readlane', 'v_cmp')):
        return _scalars(ops[0]) if ops else set()
    if '_co_' in name or 'div_scale' in name or name.startswith('v_mad_u64_u32') or name.startswith('v_mad_i64_i32'):
        return _scalars(ops[1]) if len(ops) > 1 else set()
    return set()


def too_close(assembly: str) -> list[tuple[str, str]]:
    """(writer, reader) pairs with fewer than WAIT_STATES wait states between them."""
    code = [line.split(';')[0].strip() for line in assembly.splitlines()]
    code = [x for x in code if x and not x.startswith(('.', '//')) and not x.endswith(':')]
    found = []
    for k, reader in enumerate(code):
        read = set().union(*map(_scalars, _operands(reader))) if reader.startswith(MEMORY) else set()
        waited, back = 0, k - 1
        while read and waited < WAIT_STATES and back >= 0 and not code[back].startswith(('s_branch', 's_endpgm', 's_setpc')):
            ins = code[back]
            if ins.startswith('v_') and read & _written(ins):
                found.append((ins, reader))
            waited += int(ins.split()[1], 0) + 1 if ins.startswith('s_nop') else 1
            back -= 1
    return found


def test_the_check_sees_a_short_wait():
    load = 'buffer_load_dwordx4 v1, s[12:15], s23 offen lds'
    write = 'v_readfirstlane_b32 s13, v4'
    assert too_close(f'{write}\ns_add_u32 m0, s2, 0\ns_nop 0\n{load}') == [(write, load)]
    assert too_close(f'{write}\ns_add_u32 m0, s2, 0\ns_nop 2\n{load}') == [(write, load)]
    assert too_close(f'{write}\ns_add_u32 m0, s2, 0\ns_nop 3\n{load}') == []
    assert too_close(f'{write.replace("s13", "s16")}\n{load}') == []
    carry = 'v_mad_u64_u32 v[2:3], s[22:23], v2, v4, v[6:7]'
    assert too_close(f'{carry}\n{load}') == [(carry, load)]


def _text(path: str) -> str:
    text = open(path).read()
    headers = [os.path.join(build.CSRC, h) for h in re.findall(r'#include "([^"/]+)"', text)]
    return text + ''.join(map(_text, headers))


SOURCES = [s for s in sorted(os.listdir(build.CSRC)) if s.endswith('.hip')
           and re.search(r'asm volatile\([^;]*buffer_load', _text(os.path.join(build.CSRC, s)))]


@pytest.fixture(scope='module')
def assemblies(tmp_path_factory):
    folder = tmp_path_factory.mktemp('assembly')

    def compiled(source):
        out = folder / (source + '.s')
        subprocess.run([build.HIPCC] + build.COMMON + build.FILE_FLAGS.get(source, [])
                       + ['--cuda-device-only', '-S', os.path.join(build.CSRC, source), '-o', str(out)],
                       check=True, capture_output=True)
        return out.read_text()

    with cf.ThreadPoolExecutor(max_workers=4) as pool:
        return dict(zip(SOURCES, pool.map(compiled, SOURCES)))


@pytest.mark.parametrize('source', SOURCES)
def test_resources_are_written_early_enough(source, assemblies):
    assembly = assemblies[source]
    assert assembly.count(' lds') > 0
    assert too_close(assembly) == []
