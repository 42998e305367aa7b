"""Wait states before the matrix instructions of windowed and prefixed attention, read off the assembly as
test_matrix_operand_waits.py does for the other kernels; these files are compiled side by side."""
import concurrent.futures as cf
import os
import subprocess

import pytest

from musc_hip import build

from test_matrix_operand_waits import too_close

SOURCES = [f'masked_attention_{kind}_{storage}.hip' for kind in ('window', 'prefix') for storage in ('f32', 'f16', 'bf16')]


@pytest.fixture(scope='module')
def assemblies(tmp_path_factory):
    folder = tmp_path_factory.mktemp('assembly')

    def compiled(source):
        out = folder / (source + '.s')
        subprocess.run([build.HIPCC] + build.COMMON + build.FILE_FLAGS[source]
                       + ['--cuda-device-only', '-S', os.path.join(build.CSRC, source), '-o', str(out)],
                       check=True, capture_output=True)
        return out.read_text()

    with cf.ThreadPoolExecutor(max_workers=6) as pool:
        return dict(zip(SOURCES, pool.map(compiled, SOURCES)))


@pytest.mark.parametrize('source', SOURCES)
def test_matrix_operands_are_written_early_enough(source, assemblies):
    assert assemblies[source].count('v_mfma') > 0
    assert too_close(assemblies[source]) == []
