"""What the library sets or asks once for each device of a process (csrc/per_device.h), compiled for the host."""

import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "thing_htn_2026_b200", "csrc")

PROGRAM = r"""
#include <cstdio>
#include <initializer_list>
#include "per_device.h"
#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
template <int KERNEL> int reserve(int device, int status, int* calls) {
    static OncePerDevice once;
    return once(device, [&] { ++*calls; return status; });
}
template <int KERNEL> int ask(int device, int answer, int* calls) {
    static NumberPerDevice number;
    return number(device, [&] { ++*calls; return answer; });
}
int main() {
    int calls = 0;
    CHECK(reserve<0>(0, 0, &calls) == 0 && calls == 1);
    CHECK(reserve<0>(0, 0, &calls) == 0 && calls == 1);        // once
    CHECK(reserve<0>(1, 0, &calls) == 0 && calls == 2);        // for each device
    CHECK(reserve<1>(0, 0, &calls) == 0 && calls == 3);        // and kernel
    CHECK(reserve<0>(2, 7, &calls) == 7 && calls == 4);        // what failed is tried again
    CHECK(reserve<0>(2, 0, &calls) == 0 && calls == 5);
    CHECK(reserve<0>(2, 7, &calls) == 0 && calls == 5);
    for (int beyond : {-1, 64, 1000}) {
        calls = 0;
        CHECK(reserve<0>(beyond, 0, &calls) == 0 && reserve<0>(beyond, 0, &calls) == 0 && calls == 2);
        CHECK(ask<0>(beyond, 3, &calls) == 3 && ask<0>(beyond, 4, &calls) == 4 && calls == 4);
    }
    calls = 0;
    CHECK(ask<0>(0, 20, &calls) == 20 && ask<0>(0, 9, &calls) == 20 && calls == 1);
    CHECK(ask<0>(1, 9, &calls) == 9 && ask<1>(0, 5, &calls) == 5 && calls == 3);
    CHECK(ask<0>(2, -1, &calls) == 0 && ask<0>(2, 6, &calls) == 6 && ask<0>(2, -1, &calls) == 6 && calls == 5);
    CHECK(ask<0>(3, 0, &calls) == 0 && ask<0>(3, 6, &calls) == 0 && calls == 6);      // none is an answer
    return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no C++ compiler")
def test_once_for_each_device_and_kernel(tmp_path):
    (tmp_path / "use.cpp").write_text(PROGRAM)
    done = subprocess.run(["g++", "-std=c++17", f"-I{CSRC}", str(tmp_path / "use.cpp"), "-o", str(tmp_path / "use")], capture_output=True, text=True)
    assert done.returncode == 0, done.stderr
    done = subprocess.run([str(tmp_path / "use")], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout


@pytest.mark.parametrize("name", ["mx4_pair.cu", "mx4_stream.cu"])
def test_the_4_bit_products_keep_no_other_state(name):
    """Their launches hold nothing in static variables but what is held for each device."""
    with open(os.path.join(CSRC, name)) as handle:
        lines = [line.strip() for line in handle if line.startswith("    static ") and "constexpr" not in line and "static_assert" not in line]
    assert all(line.startswith("static NumberPerDevice") for line in lines), lines
