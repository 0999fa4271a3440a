"""Without the reference's sources its library is not built; tests that compare with it are skipped, not failed."""
import os
import subprocess
import sys

import pytest

import oracle
from conftest import ROOT

INNER = '''
import oracle

def test_compares_with_the_reference():
    oracle.Reference(path="{path}")

def test_opens_something_else():
    open("{path}")
'''


def test_the_error_says_what_is_missing(tmp_path):
    with pytest.raises(oracle.ReferenceMissing, match="make -C oracle ref"):
        oracle.Reference(path=str(tmp_path / "none.so"))


def test_such_a_test_is_skipped(tmp_path):
    (tmp_path / "test_inner.py").write_text(INNER.format(path=tmp_path / "none.so"))
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([os.path.join(ROOT, "tests"), ROOT]))
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-rs", "-p", "conftest", "-p", "no:cacheprovider", str(tmp_path)],
                       capture_output=True, text=True, env=env, cwd=tmp_path, timeout=300)
    assert "1 failed, 1 skipped" in r.stdout and "test_opens_something_else" in r.stdout, r.stdout + r.stderr
