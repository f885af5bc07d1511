"""Argument checks of the paged cache's C entry points that need no device, and the sign generator."""
import ctypes as C

import numpy as np
import pytest

from oracle import loader


@pytest.fixture(scope="module")
def lib():
    from adaptq_b200 import build
    build.build_library()
    import adaptq_b200
    return adaptq_b200.load()


def desc(**change):
    from adaptq_b200 import _lib
    # addresses that no call below follows
    d = dict(k_pages=4096, v_pages=8192, k_scales=4096, v_scales=8192, signs=4096, status=4096, n_pages=4, n_kv_heads=2, page_size=16,
             dim=64, k_bits=4, v_bits=4, device=0)
    d.update(change)
    return _lib.Paged(*[d[f] for f, _ in _lib.Paged._fields_])


def rotary(**change):
    from adaptq_b200 import _lib
    d = dict(turns=4096, factor=1.0, dim=64, interleaved=0)
    d.update(change)
    return _lib.RotaryDesc(*[d[f] for f, _ in _lib.RotaryDesc._fields_])


def append(lib, d, type=0, n_seqs=1, n_tokens=1, k=4096, rot=None, width=1):
    return lib.adaptq_paged_append(C.addressof(d) if d else None, k, 128, 64, 4096, 128, 64, type, 4096, 1, width, 4096, 0, None, n_seqs,
                                   n_tokens, C.addressof(rot) if rot else None, None)


def attend(lib, d, heads=4, scale=0.125, n_seqs=1, q=4096, size=1 << 30, type=0):
    return lib.adaptq_paged_attend(C.addressof(d), q, 256, 64, 4096, 256, 64, type, 4096, 1, 1, 4096, n_seqs, heads, C.c_float(scale), None, 4096,
                                   size, None)


@pytest.mark.parametrize("change,text", [
    (dict(k_pages=None), "null pointer"), (dict(status=None), "null pointer"), (dict(signs=None), "null pointer"), (dict(dim=32), "dimension"),
    (dict(dim=257), "dimension"), (dict(k_bits=1), "bits"), (dict(v_bits=16), "bits"), (dict(page_size=24), "page_size"), (dict(n_pages=0), "pages"),
    (dict(n_pages=1 << 31), "pages"), (dict(n_kv_heads=0), "heads"), (dict(k_pages=4104), "aligned"), (dict(v_scales=8196), "aligned")])
def test_bad_caches(lib, change, text):
    d = desc(**change)
    for call in (append, attend):
        assert call(lib, d) == -1
        assert text in lib.adaptq_last_error().decode()


def test_bad_calls(lib):
    err = lambda: lib.adaptq_last_error().decode()  # noqa: E731
    d = desc()
    assert append(lib, None) == -1 and "null cache" in err()
    assert append(lib, d, type=3) == -1 and "type" in err()
    assert append(lib, d, n_tokens=-1) == -1 and "negative" in err()
    assert append(lib, d, k=None) == -1 and "null pointer" in err()
    assert append(lib, d, n_tokens=1 << 40) == -1 and "too many" in err()
    for bad in (dict(turns=None), dict(dim=63), dict(dim=66), dict(dim=0)):
        assert append(lib, d, rot=rotary(**bad)) == -1 and "rotary" in err()
    assert append(lib, d, n_tokens=0) == 0 and append(lib, d, n_seqs=0) == 0
    assert attend(lib, d, heads=3) == -1 and "multiple" in err()
    assert attend(lib, d, heads=0) == -1 and "multiple" in err()
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert attend(lib, d, scale=scale) == -1 and "scale" in err()
    assert attend(lib, d, q=None) == -1 and "null pointer" in err()
    assert attend(lib, d, size=0) == -1 and "workspace" in err()
    assert attend(lib, d, n_seqs=0) == 0
    assert append(lib, d, k=4097) == -1 and "aligned" in err()
    assert append(lib, d, k=4098, type=0) == -1 and "aligned" in err()
    assert attend(lib, d, q=4097, type=2) == -1 and "aligned" in err()
    assert append(lib, desc(status=4098)) == -1 and "aligned" in err()
    assert append(lib, d, rot=rotary(turns=4100)) == -1 and "rotary" in err()
    r = rotary()
    args = lambda **k: [C.addressof(k.get("r", r)), k.get("x", 4096), 64, 64, 4096, 64, 64, k.get("type", 0), 4096, 0, k.get("n", 1), k.get("h", 1),  # noqa: E731
                        k.get("dim", 64), 0, 0, None]
    for bad in (dict(x=None), dict(x=4097), dict(x=4098), dict(type=7), dict(n=-1), dict(h=-1), dict(dim=0), dict(dim=62), dict(r=rotary(dim=3))):
        assert lib.adaptq_rotary_apply(*args(**bad)) == -1 and err()
    assert lib.adaptq_rotary_apply(*args(n=0)) == 0


def test_signs_are_those_of_the_rings(lib):
    orc = loader.oracle()
    for seed, heads, dim in ((42, 3, 64), (0, 2, 100), (2**64 - 1, 2, 256)):
        p = 64 if dim <= 64 else 128 if dim <= 128 else 256
        words = np.zeros((heads, p // 32), np.uint32)
        assert lib.adaptq_paged_signs(C.c_uint64(seed), heads, dim, words.ctypes.data) == 0
        for h in range(heads):
            want = loader.Head(orc, dim, 4, 4, 4, loader.mha_head_seed(seed, h), 0.0, 0).signs()
            got = 1 - 2 * ((words[h][:, None] >> np.arange(32, dtype=np.uint32)) & 1).astype(np.int8).reshape(-1)
            assert (got == want).all()
    assert lib.adaptq_paged_signs(C.c_uint64(1), 1, 32, words.ctypes.data) == -1
    assert lib.adaptq_paged_signs(C.c_uint64(1), 1, 64, None) == -1


def test_take_status_refusals(lib):
    err = lambda: lib.adaptq_last_error().decode()  # noqa: E731
    d = desc()
    assert lib.adaptq_paged_take_status(None, 4096, None) == -1 and "null cache" in err()
    assert lib.adaptq_paged_take_status(C.addressof(d), None, None) == -1 and "null pointer" in err()
    assert lib.adaptq_paged_take_status(C.addressof(d), 4098, None) == -1 and "aligned" in err()
    d = desc(status=None)
    assert lib.adaptq_paged_take_status(C.addressof(d), 4096, None) == -1 and "null pointer" in err()
