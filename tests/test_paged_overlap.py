"""What the paged operators and the draft verification write must not overlap:
the host-side test of two strided views against plain enumeration, and the C
ABI's refusals (every call here is refused before it reaches a GPU)."""

import ctypes
import itertools
import random
import shutil
import subprocess

import pytest
import torch

import capi_lib
from test_native_build import built  # noqa: F401  (fixture)
from test_paged import FAKE, Rows, _cache
from test_paged import lib as capi  # noqa: F401  (fixture)

OVERLAP = 9
FAR = 1 << 40  # another place, never dereferenced


@pytest.fixture
def lib(capi):  # noqa: F811
    if torch.cuda.is_available():
        pytest.skip("addresses that nothing is behind: only where no GPU could follow them")
    return capi


# ------------------------------------------------------------ strided views --
@pytest.fixture(scope="module")
def views(tmp_path_factory):
    d = tmp_path_factory.mktemp("overlap")
    (d / "v.cpp").write_text("""
#include "overlap.h"
using namespace persona::overlap;
static View view(const int64_t* a) { return View{reinterpret_cast<void*>(a[0]), a[1], {a[2], a[3], a[4]}, {a[5], a[6], a[7]}}; }
extern "C" int is_nested(const int64_t* a) { return nested(view(a)); }
extern "C" int do_share(const int64_t* a, const int64_t* b) { return share(view(a), view(b)); }
extern "C" int do_ranges(const int64_t* a, const int64_t* b) { return ranges_meet(view(a), view(b)); }
""")
    subprocess.run([shutil.which("g++"), "-std=c++17", "-O1", "-shared", "-fPIC", "-I",
                    str(capi_lib.ROOT / "multi-lora-llm-kernel_b200" / "csrc"), str(d / "v.cpp"), "-o", str(d / "v.so")], check=True)
    return ctypes.CDLL(str(d / "v.so"))


def _c(view):
    p, inner, size, stride = view
    return (ctypes.c_int64 * 8)(p, inner, *size, *stride)


def _bytes(view):
    """Every byte the view reaches, one entry each time."""
    p, inner, size, stride = view
    return [p + sum(i * s for i, s in zip(ix, stride)) + x for ix in itertools.product(*map(range, size)) for x in range(inner)]


def test_views_against_enumeration(views):
    rng = random.Random(1)
    seen = {k: 0 for k in ("twice", "once", "meet", "apart", "near")}
    for _ in range(20000):
        inner = rng.randint(1, 4)
        size = [rng.randint(1, 3) for _ in range(3)]
        stride = [rng.randint(0, 40) for _ in range(3)]
        if rng.random() < 0.6:  # as slices and transposes of a buffer have them
            at, order = inner, [0, 1, 2]
            rng.shuffle(order)
            for i in order:
                stride[i] = at + rng.randint(0, 3)
                at = stride[i] * size[i]
        a = (1000, inner, size, stride)
        reached = _bytes(a)
        once = len(set(reached)) == len(reached)
        if views.is_nested(_c(a)):
            assert once  # what is taken for apart is
            seen["once"] += 1
        else:
            seen["twice"] += not once
        sizes = [n if rng.random() < 0.5 else rng.randint(1, 3) for n in size]
        strides = [s if rng.random() < 0.8 else rng.randint(0, 40) for s in stride]
        b = (1000 + rng.randint(-90, 90), inner if rng.random() < 0.8 else rng.randint(1, 4), sizes, strides)
        meet = bool(set(reached) & set(_bytes(b)))
        if meet:
            assert views.do_share(_c(a), _c(b)) and views.do_ranges(_c(a), _c(b))
            seen["meet"] += 1
        elif not views.do_share(_c(a), _c(b)):
            seen["apart"] += 1
            seen["near"] += views.do_ranges(_c(a), _c(b))  # told apart inside one another
        elif strides == stride and sizes == size and views.is_nested(_c(a)) and b[1] == inner:
            raise AssertionError(f"alike and apart, taken for shared: {a} {b}")
    assert min(seen.values()) > 200, seen


def test_views_of_large_strides_and_of_nothing(views):
    big = (1 << 20, 256, [1 << 31, 1024, 64], [1 << 60, 1 << 40, 256])
    assert views.is_nested(_c(big)) and views.do_share(_c(big), _c(big))
    assert not views.do_share(_c(big), _c(((1 << 20) + 64 * 256, 256, *big[2:])))
    none = (1 << 20, 256, [0, 4, 4], [1024, 256, 0])
    assert not views.do_share(_c(none), _c(big)) and not views.do_ranges(_c(big), _c(none))


# ------------------------------------------------------------------- C ABI --
PAGES = 9 * 8 * 16 * 128 * 2  # bytes of one cache of _cache()


def _kv(**change):
    """k and v caches of _cache() apart from each other and from the index arrays."""
    c = dict(k=FAR, v=FAR + PAGES)
    c.update(change)
    return _cache(**c)


def _e4m3(**change):
    return _kv(kind=1, k_scale=FAR + (1 << 30), v_scale=FAR + (1 << 31), **change)


Q, QO, K, V = (Rows(2 * FAR + i * (1 << 24), h * 128, 128) for i, h in enumerate((32, 32, 8, 8)))


def _write(lib, cache, q=Q, q_out=QO, k=K, v=V, rows=4):
    r = ctypes.byref
    return lib.persona_paged_rope_cache(r(cache), r(q), r(q_out), r(k), r(v), rows, 32, 1e6, 0, None, None)


def test_write_refuses_caches_that_overlap(lib):
    for cache in (_kv(v=FAR),                                                      # k and v the same
                  _kv(v=FAR + 128 * 2), _kv(v=FAR + PAGES - 16),
                  _kv(page_stride=128, head_stride=16 * 128),                      # pages in one another
                  _kv(page_stride=0), _kv(head_stride=0), _kv(head_stride=15 * 128), _kv(page_stride=8 * 16 * 128 - 8),
                  _e4m3(scale_page_stride=0), _e4m3(scale_head_stride=0), _e4m3(scale_head_stride=15),
                  _kv(page_table=FAR + 64), _kv(lengths=FAR + PAGES + 8), _kv(indptr=FAR)):
        assert _write(lib, cache) == OVERLAP
    same = _e4m3()
    same.v_scale = same.k_scale
    assert _write(lib, same) == OVERLAP
    same.v_scale = same.k_scale + 4 * 16
    assert _write(lib, same) == OVERLAP


def test_write_refuses_rows_that_overlap(lib):
    at = lambda p, row=4096, head=128: Rows(p, row, head)  # noqa: E731
    assert _write(lib, _kv(), q_out=at(QO.p, row=128)) == OVERLAP    # rows in one another
    assert _write(lib, _kv(), q_out=at(QO.p, head=0)) == OVERLAP
    assert _write(lib, _kv(), q_out=at(Q.p + 256)) == OVERLAP        # one head on
    assert _write(lib, _kv(), q=K, q_out=at(K.p), k=at(K.p)) == OVERLAP
    assert _write(lib, _kv(), q_out=at(V.p + 2 * 128 * 7)) == OVERLAP
    for p in (FAR, FAR + PAGES + 1024):                              # inside the pages
        assert _write(lib, _kv(), q_out=at(p)) == OVERLAP
        assert _write(lib, _kv(), q=at(p), q_out=QO) == OVERLAP
        assert _write(lib, _kv(), k=at(p)) == OVERLAP and _write(lib, _kv(), v=at(p)) == OVERLAP
    assert _write(lib, _e4m3(), q_out=at(FAR + (1 << 30))) == OVERLAP  # the scales
    assert _write(lib, _kv(page_table=QO.p + 64)) == OVERLAP


def test_read_and_attention_refuse_outputs_that_overlap(lib):
    r = ctypes.byref
    read = lambda c, k, v: lib.persona_paged_cache_read(r(c), r(k), r(v), 4, 0, None, None)  # noqa: E731
    row = lambda p, step=1024: Rows(p, step, 128)  # noqa: E731
    assert read(_kv(), K, K) == OVERLAP and read(_kv(), K, row(K.p + 128 * 2)) == OVERLAP
    assert read(_kv(), row(FAR), V) == OVERLAP and read(_kv(), K, row(FAR + PAGES)) == OVERLAP
    assert read(_kv(), row(K.p, 128), V) == OVERLAP and read(_e4m3(), K, row(FAR + (1 << 31))) == OVERLAP
    assert read(_kv(lengths=K.p), K, V) == OVERLAP
    ws = 4 * FAR

    def attend(cache=None, q=Q, out=QO, ws=ws):
        return lib.persona_paged_attention(r(cache or _kv()), r(q), r(out), 4, 32, 0.1, 0, 1, 0, ws, 1 << 40, None, None)

    assert attend(out=Q) == OVERLAP and attend(out=Rows(Q.p + 256, 4096, 128)) == OVERLAP
    assert attend(out=Rows(FAR, 4096, 128)) == OVERLAP and attend(out=Rows(QO.p, 2048, 128)) == OVERLAP
    assert attend(cache=_kv(indptr=QO.p + 4)) == OVERLAP
    for inside in (Q.p, QO.p, FAR, FAR + PAGES, FAKE):
        assert attend(ws=inside) == OVERLAP


def test_verification_refuses_outputs_that_overlap(lib):
    place = {n: FAR + i * (1 << 24) for i, n in enumerate(("target", "draft", "d", "ip", "ua", "us", "out", "acc"))}

    def call(**change):
        a = dict(place, **change)
        return lib.persona_verify_draft(a["target"], 100, a["draft"], 100, 2, a["d"], a["ip"], a["ua"], a["us"], a["out"],
                                        a["acc"], 3, 2, 100, None, None)

    for name in ("target", "draft", "d", "ip", "ua", "us", "acc"):
        assert call(out=place[name]) == OVERLAP
    for name in ("target", "draft", "d", "ip", "ua", "us", "out"):
        assert call(acc=place[name]) == OVERLAP
    assert call(out=place["d"] + 16) == OVERLAP and call(acc=place["ip"] + 8) == OVERLAP
    assert call(out=place["target"] + 2 * 400 + 392) == OVERLAP  # the last row's last element
    assert b"overlaps" in _string(lib, OVERLAP)


def _string(lib, status):
    lib.persona_status_string.restype = ctypes.c_char_p
    return lib.persona_status_string(status)
