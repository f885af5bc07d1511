"""When the build compiles a translation unit anew (a stand-in for the compiler, no device needed)."""
import os
import subprocess
import sys
import threading

import pytest

STAND_IN = '''#!{python}
import os, sys, time
out = sys.argv[sys.argv.index("-o") + 1]
with open(os.environ["STAND_IN_LOG"], "a") as f:
    f.write(os.path.basename(out) + "\\n")
time.sleep(float(os.environ.get("STAND_IN_SECONDS", "0")))
if os.path.exists(out + ".busy"):
    sys.exit("two compilers at once")
open(out + ".busy", "w").close()
open(out, "w").write("built")
if "-MF" in sys.argv:
    src = sys.argv[-1]
    open(sys.argv[sys.argv.index("-MF") + 1], "w").write(out + ": " + src + " " + os.path.join(os.path.dirname(src), "a.cuh") + " \\\\\\n /usr/include/x.h\\n")
time.sleep(float(os.environ.get("STAND_IN_SECONDS", "0")))
os.remove(out + ".busy")
'''


@pytest.fixture()
def tree(tmp_path, monkeypatch):
    """A copy of build.py over two small units; calls of the compiler are written to a log."""
    import adaptq_b200
    package = tmp_path / "one" / "adaptq_b200"
    (package / "csrc").mkdir(parents=True)
    (tmp_path / "one" / "include").mkdir()
    with open(os.path.join(os.path.dirname(adaptq_b200.__file__), "build.py")) as f:
        text = f.read()
    (package / "build.py").write_text(text)
    for name in ("adaptq_b200.cu", "paged.cu", "a.cuh"):
        (package / "csrc" / name).write_text("x")
    (tmp_path / "nvcc").write_text(STAND_IN.format(python=sys.executable))
    (tmp_path / "nvcc").chmod(0o755)
    monkeypatch.setenv("PATH", f"{tmp_path}:{os.environ['PATH']}")
    monkeypatch.setenv("STAND_IN_LOG", str(tmp_path / "log"))
    return tmp_path


def age(root):
    """Everything that is there becomes ten seconds older."""
    for folder, _, names in os.walk(root):
        for n in names:
            t = os.path.getmtime(os.path.join(folder, n)) - 10
            os.utime(os.path.join(folder, n), (t, t))


def build(root, log):
    log.write_text("")
    subprocess.check_call([sys.executable, "-c", "import build; build.UNITS = [('adaptq_b200.cu', 'adaptq_b200', []), ('paged.cu', 'paged', [])]; "
                           "build.build_library()"], cwd=root / "adaptq_b200")
    return sorted(log.read_text().split())


EVERYTHING = ["adaptq_b200.o", "libadaptq_b200.so", "paged.o"]


def test_units_are_compiled_when_their_sources_change(tree):
    one, log = tree / "one", tree / "log"
    assert build(one, log) == EVERYTHING
    assert build(one, log) == []
    age(one)
    (one / "adaptq_b200" / "csrc" / "paged.cu").write_text("y")
    assert build(one, log) == ["libadaptq_b200.so", "paged.o"]
    age(one)
    (one / "adaptq_b200" / "csrc" / "a.cuh").write_text("y")
    assert build(one, log) == EVERYTHING


def test_a_tree_that_was_moved_is_compiled_anew(tree):
    """The compiler's lists name files of the old place: nothing tells that the objects are up to date."""
    one, log = tree / "one", tree / "log"
    build(one, log)
    two = tree / "two"
    os.rename(one, two)
    age(two)
    (two / "adaptq_b200" / "csrc" / "paged.cu").write_text("y")
    assert "paged.o" in build(two, log)
    os.symlink(two, tree / "three")   # another name of the same place is no move
    age(two)
    (two / "adaptq_b200" / "csrc" / "paged.cu").write_text("z")
    assert build(tree / "three", log) == ["libadaptq_b200.so", "paged.o"]


def test_other_flags_compile_anew(tree):
    one, log = tree / "one", tree / "log"
    build(one, log)
    age(one)
    path = one / "adaptq_b200" / "build.py"
    path.write_text(path.read_text().replace('"-O3"', '"-O2"'))
    assert build(one, log) == EVERYTHING


def test_two_builds_at_once(tree, monkeypatch):
    """The second waits for the first and finds nothing left to do."""
    one, log = tree / "one", tree / "log"
    monkeypatch.setenv("STAND_IN_SECONDS", "0.3")
    failed = []

    def run():
        try:
            subprocess.check_call([sys.executable, "-c", "import build; build.UNITS = [('adaptq_b200.cu', 'adaptq_b200', []), ('paged.cu', 'paged', [])]; "
                                   "build.build_library()"], cwd=one / "adaptq_b200")
        except subprocess.CalledProcessError as e:
            failed.append(e)

    threads = [threading.Thread(target=run) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    assert sorted(log.read_text().split()) == EVERYTHING
