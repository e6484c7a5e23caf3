"""The bookkeeping of a cache's pages (csrc/page_book.h), on the CPU (tests/cpp/page_book_test.cpp)."""
import os
import subprocess

import pytest

SRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "page_book_test.cpp")


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("page_book") / "page_book_test")
    r = subprocess.run([os.environ.get("CXX", "g++"), "-std=c++17", "-O1", "-Wall", "-Wextra", "-D_GLIBCXX_ASSERTIONS", SRC, "-o", exe],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return exe


@pytest.mark.parametrize("check", ["random", "refusals", "branches"])
def test_page_book(program, check):
    r = subprocess.run([program, check], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr


def test_pages_in_common(program):
    r = subprocess.run([program, "common"], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
