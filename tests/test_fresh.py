"""Which products may request their weights early (csrc/fresh.cuh, compiled by the host compiler)."""
import ctypes
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(__file__), os.pardir, "metaltile_b200", "csrc")


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("fresh")
    src = d / "fresh.cpp"
    src.write_text('#include "fresh.cuh"\nusing mtc::FreshWeights;\nextern "C" {\n'
                   "void *make() { return new FreshWeights; }\n"
                   "void done(void *f) { delete static_cast<FreshWeights *>(f); }\n"
                   "void written(void *f, long s, int c) { static_cast<FreshWeights *>(f)->written(reinterpret_cast<void *>(s), c); }\n"
                   "int known(void *f) { return static_cast<FreshWeights *>(f)->known(); }\n"
                   "int early(void *f, long s, int c) { return static_cast<FreshWeights *>(f)->early(reinterpret_cast<void *>(s), c); }\n"
                   "}\n")
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", CSRC, str(src), "-o", str(d / "fresh.so"), "-lpthread"], check=True)
    so = ctypes.CDLL(str(d / "fresh.so"))
    so.make.restype = ctypes.c_void_p
    return so


@pytest.fixture
def fresh(lib):
    f = ctypes.c_void_p(lib.make())

    class Fresh:
        def written(self, stream, captured=False):
            lib.written(f, ctypes.c_long(stream), int(captured))

        def early(self, stream, captured=False):
            return not lib.known(f) or bool(lib.early(f, ctypes.c_long(stream), int(captured)))

        def known(self):
            return bool(lib.known(f))

    yield Fresh()
    lib.done(f)


def test_the_first_product_behind_a_quantizer_waits_and_the_next_does_not(fresh):
    assert fresh.early(1) and not fresh.known()
    fresh.written(1)
    fresh.written(1)
    assert fresh.early(2) and not fresh.early(1) and fresh.early(1) and not fresh.known()


def test_a_captured_product_leaves_the_wait_to_one_that_runs(fresh):
    fresh.written(1)
    assert fresh.early(1, captured=True) and not fresh.early(1) and fresh.early(1)
    fresh.written(1, captured=True)
    assert not fresh.early(1, captured=True) and fresh.early(1, captured=True)


def test_captured_quantizers_without_products_cost_what_runs_nothing(fresh):
    for s in range(200):
        fresh.written(s, captured=True)
    for s in range(64):
        fresh.written(1000 + s)
    assert all(fresh.early(s) for s in range(200))
    assert not any(fresh.early(1000 + s) for s in range(64)) and all(fresh.early(1000 + s) for s in range(64))
    assert not fresh.early(300, captured=True)               # more captures than were kept apart: none of theirs starts early


def test_more_streams_than_the_list_holds_start_no_product_early(fresh):
    for s in range(65):
        fresh.written(s)
    assert not any(fresh.early(s) for s in range(65)) and not fresh.early(7)


def test_a_capture_that_is_over_leaves_nothing(fresh):
    for s in range(500):                                     # one stream after another: captured on, then used
        fresh.written(s, captured=True)
        assert fresh.early(s)
    assert not fresh.known() and fresh.early(3, captured=True)
