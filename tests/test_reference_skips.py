"""Which tests are skipped where the reference's sources are missing, and that no other is."""
import os
import subprocess
import sys

import pytest

import conftest
import oracle

TESTS = os.path.dirname(os.path.abspath(__file__))


def run(tmp_path, text, **env):
    (tmp_path / "test_it.py").write_text(text)
    e = dict(os.environ, PYTHONPATH=TESTS, **env)
    return subprocess.run([sys.executable, "-m", "pytest", "-q", "-p", "conftest", "-p",
                           "no:cacheprovider", "--rootdir", str(tmp_path), str(tmp_path)],
                          capture_output=True, text=True, timeout=120, env=e, cwd=tmp_path)


def test_an_oracle_that_is_not_built_fails_the_test(tmp_path):
    r = run(tmp_path, "import oracle\n\n\ndef test_other():\n"
                      "    raise oracle.ReferenceNotBuilt('not built')\n")
    assert r.returncode == 1 and "1 failed" in r.stdout, r.stdout


@pytest.mark.skipif(oracle.ref_available(), reason="the reference's library is there")
@pytest.mark.parametrize("sources", [False, True])
def test_comparisons_are_skipped_only_without_sources(tmp_path, sources):
    """With the sources at hand a library that was not built is a failure, not a skip."""
    tree = tmp_path / "reference"
    tree.mkdir()
    if sources:
        (tree / "fused_winograd.c").write_text("")
    name = sorted(conftest.NEEDS_REFERENCE)[0]
    r = run(tmp_path, f"import oracle\n\n\ndef {name}():\n    oracle.ref()\n",
            CWG_REFERENCE=str(tree))
    assert ("1 failed" if sources else "1 skipped") in r.stdout, r.stdout
