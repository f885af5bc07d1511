"""The paged cache's and the rotation's tests under the checked build (libadaptq_b200_checked.so), in a child process: there an
index check stands in front of every store into pages, outputs and workspace and every read of rows, pages and tables;
one that fails skips the access and leaves a bit in the status word, which tests/paged_checked_plugin.py looks at after
every test."""
import os
import subprocess
import sys

import pytest

from test_gpu_checked_build import CHECKED, ROOT

pytestmark = pytest.mark.gpu


def test_paged_suites_pass_under_the_checked_build(gpu_lib):
    if not os.path.exists(CHECKED):
        pytest.skip("libadaptq_b200_checked.so not built (python -m adaptq_b200.build --checked)")
    env = dict(os.environ, ADAPTQ_B200_LIB=CHECKED, PYTHONPATH=os.pathsep.join([ROOT, os.path.join(ROOT, "tests"), os.environ.get("PYTHONPATH", "")]))
    probe = subprocess.run([sys.executable, "-c", "import adaptq_b200; print(adaptq_b200.load().adaptq_version().decode())"],
                           capture_output=True, text=True, env=env, cwd=ROOT, timeout=300)
    assert probe.stdout.strip().endswith("-sm100a-checked"), probe.stdout + probe.stderr
    files = [os.path.join("tests", f) for f in ("test_gpu_paged.py", "test_gpu_paged_calls.py", "test_gpu_paged_runs.py", "test_gpu_paged_precision.py")]
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-x", "-m", "gpu", "-p", "no:cacheprovider", "-p", "paged_checked_plugin", *files],
                       capture_output=True, text=True, env=env, cwd=ROOT, timeout=3000)
    assert r.returncode == 0, r.stdout[-6000:] + r.stderr[-2000:]


def test_a_failed_check_is_reported(gpu_lib, tmp_path):
    """The word's bit, set from outside (no kernel is made to fail one): check() raises, and the plugin fails the test."""
    from adaptq_b200 import PagedKVCache
    cache = PagedKVCache(1, 1, 64, page_size=16)
    cache._status.fill_(256)
    with pytest.raises(RuntimeError, match="index check"):
        cache.check()
    cache.check()
    (tmp_path / "test_bit.py").write_text("def test_bit():\n    from adaptq_b200 import PagedKVCache\n    c = PagedKVCache(1, 1, 64, page_size=16)\n"
                                          "    c._status.fill_(256)\n\n\ndef test_clean():\n    from adaptq_b200 import PagedKVCache\n"
                                          "    PagedKVCache(1, 1, 64, page_size=16)\n")
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([ROOT, os.path.join(ROOT, "tests"), os.environ.get("PYTHONPATH", "")]))
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-p", "no:cacheprovider", "-p", "paged_checked_plugin", str(tmp_path)],
                       capture_output=True, text=True, env=env, cwd=tmp_path, timeout=600)
    assert "a device-side index check failed" in r.stdout and "1 failed, 1 passed" in r.stdout, r.stdout[-3000:] + r.stderr[-1000:]
