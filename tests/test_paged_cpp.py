"""PagedKVCache (include/paged_kv_cache.hpp) and the launchers of
include/kernels/paged_kernels.hpp: the headers compile as C++23 and C++17, and the test
program tests/cpp/test_paged_cache.cpp, built against the library, passes on the GPU."""
import pathlib
import subprocess

import pytest

ROOT = pathlib.Path(__file__).resolve().parents[1]
BIN = ROOT / "tests" / "cpp" / "_build" / "test_paged_cache"


@pytest.mark.parametrize("std", ["c++17", "c++23"])
def test_headers_compile(tmp_path, std):
    src = tmp_path / "use_headers.cpp"
    src.write_text(
        '#include "paged_kv_cache.hpp"\n'
        "struct Cfg { size_t num_layers = 2, num_heads = 8, num_kv_heads = 4, head_dim = 128; };\n"
        "void f(const int32_t* d) { PagedKVCache c{Cfg{}, 8, 16, 2, 4}; c.grow(d); c.compact(); }\n")
    r = subprocess.run(["/opt/rocm/bin/hipcc", f"-std={std}", "-fsyntax-only", "-I",
                        str(ROOT / "include"), str(src)], capture_output=True, text=True,
                       timeout=120)
    assert r.returncode == 0, r.stderr


@pytest.mark.gpu
def test_paged_cache_program(gpu):
    assert BIN.exists(), "tests/cpp is not built"
    r = subprocess.run([str(BIN)], capture_output=True, text=True, timeout=100)
    print(r.stdout, r.stderr)
    assert r.returncode == 0 and "FAIL" not in r.stdout
    assert r.stdout.count("PASS") == 7
