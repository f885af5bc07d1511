"""Compile the CUDA library in-tree: adaptq_b200/libadaptq_b200.so (sm_100a only)."""
from __future__ import annotations

import fcntl
import os
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor

_THIS = os.path.abspath(__file__)
_HERE = os.path.dirname(_THIS)
# translation units: source, name of the object, defines
UNITS = [("adaptq_b200.cu", "adaptq_b200", []), ("paged.cu", "paged", [])] + \
        [("paged_attend.cu", f"paged_attend_k{k}v{v}", [f"-DAQ_KB={k}", f"-DAQ_VB={v}"]) for k in (4, 3, 2) for v in (4, 3, 2)]
OBJ = os.path.join(_HERE, "obj")
LIB = os.path.join(_HERE, "libadaptq_b200.so")
# the same sources with -DADAPTQ_CHECKED: device-side index checks that record a status
# instead of trapping, guard bytes behind every device buffer (see csrc/common.cuh)
LIB_CHECKED = os.path.join(_HERE, "libadaptq_b200_checked.so")


def _nvcc() -> str:
    for cand in (shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found; the AdapTQ B200 library cannot be built")


def sources():
    d = os.path.join(_HERE, "csrc")
    inc = os.path.join(os.path.dirname(_HERE), "include")
    return [os.path.join(d, f) for f in sorted(os.listdir(d))] + \
           [os.path.join(inc, f) for f in sorted(os.listdir(inc))] + [_THIS]  # flags and units


def is_stale(lib: str = LIB) -> bool:
    if not os.path.exists(lib):
        return True
    t = os.path.getmtime(lib)
    return any(os.path.getmtime(s) > t for s in sources())


def _object_is_stale(obj: str, src: str) -> bool:
    """Older than this file or anything of this tree that its translation unit includes (from the compiler's list, which
    tells nothing if it was made for a tree of another place: then `src` is not in it)."""
    dep = obj + ".d"
    if not (os.path.exists(obj) and os.path.exists(dep)):
        return True
    with open(dep) as f:
        names = f.read().replace("\\\n", " ").split(":", 1)[1].split()
    root, t = os.path.realpath(os.path.dirname(_HERE)) + os.sep, os.path.getmtime(obj)
    mine = [n for n in map(os.path.realpath, names) if n.startswith(root)]
    return os.path.realpath(src) not in mine or any(not os.path.exists(n) or os.path.getmtime(n) > t for n in [*mine, _THIS])


def build_library(force: bool = False, verbose: bool = False, checked: bool = False) -> str:
    """nvcc -gencode arch=compute_100a,code=sm_100a ... -> libadaptq_b200.so
    (checked=True: libadaptq_b200_checked.so, compiled with -DADAPTQ_CHECKED).  The translation
    units are compiled side by side."""
    lib = LIB_CHECKED if checked else LIB
    if not force and not is_stale(lib):
        return lib
    os.makedirs(OBJ, exist_ok=True)
    with open(os.path.join(OBJ, "lock"), "w") as lock:  # one build at a time: they share the objects
        fcntl.flock(lock, fcntl.LOCK_EX)
        if force or is_stale(lib):
            _compile_and_link(lib, force, verbose, checked)
    return lib


def _compile_and_link(lib, force, verbose, checked):
    arch = ["-gencode", "arch=compute_100a,code=sm_100a"]
    flags = [*arch, "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC", "-diag-suppress", "1886"]
    if checked:
        flags.append("-DADAPTQ_CHECKED=1")
    if verbose:
        flags += ["-Xptxas", "-v"]

    def compile_unit(unit):
        name, src = unit[1], os.path.join(_HERE, "csrc", unit[0])
        obj = os.path.join(OBJ, name + (".checked.o" if checked else ".o"))
        if force or _object_is_stale(obj, src):
            subprocess.check_call([_nvcc(), *flags, *unit[2], "-MD", "-MF", obj + ".d", "-c", "-o", obj, src])
        return obj

    with ThreadPoolExecutor(os.cpu_count() or 1) as pool:
        objects = list(pool.map(compile_unit, UNITS))
    subprocess.check_call([_nvcc(), *arch, "-Xcompiler", "-fPIC", "-shared", "-o", lib, *objects])


if __name__ == "__main__":
    import sys
    print(build_library(force=True, verbose=True, checked="--checked" in sys.argv))
