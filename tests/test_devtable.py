"""The launch-table cache (csrc/devtable.h) on the CPU, over a runtime that only
keeps books (tests/fixtures/devtable): a table is written before anything reads it,
whichever stream or capture met it first."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which('g++') is None, reason='needs a host compiler')
def test_a_table_is_written_before_it_is_read(tmp_path):
    shutil.copy(os.path.join(ROOT, 'csrc', 'devtable.h'), str(tmp_path))
    for name in ('common.h', 'main.cpp'):
        shutil.copy(os.path.join(ROOT, 'tests', 'fixtures', 'devtable', name), str(tmp_path))
    exe = str(tmp_path / 'devtable')
    subprocess.run(['g++', '-std=c++17', '-O1', '-pthread', '-o', exe, str(tmp_path / 'main.cpp')],
                   check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout
