"""Numbers of tokens that a branch is made with, on the CPU (tests/cpp/page_book_fork_test.cpp)."""
import os
import subprocess

SRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "page_book_fork_test.cpp")


def test_tokens_of_a_branch(tmp_path):
    exe = str(tmp_path / "page_book_fork_test")
    r = subprocess.run([os.environ.get("CXX", "g++"), "-std=c++17", "-O1", "-Wall", "-Wextra", "-D_GLIBCXX_ASSERTIONS", SRC, "-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr
