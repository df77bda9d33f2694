"""CPU tests of which form a product on 8-bit integers takes: every size has one, and the sizes of the GPU tests have
the forms that they are there for, with more steps than stages."""
import os
import subprocess
import sys

import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from int8_shapes import DEEP, FORMS  # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def exe(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("forms")
    (tmp / "forms.cpp").write_text(r'''
#include <stdio.h>
#include "icua_int8.h"
using namespace icua;
int main(int argc, char**) {
    if (argc > 1) {
        const int sizes[] = {1, 2, 15, 16, 17, 31, 64, 127, 128, 129, 255, 1000, 4096, 1 << 16, 1 << 22, 1 << 24}, deep[] = {16, 128, 2048, 2064, 6144, 1 << 17};
        for (int gated = 0; gated < 2; ++gated)
            for (int m : sizes)
                for (int n : sizes)
                    for (int k : deep) {
                        if ((long long)m * n > 1LL << 36 || n > 1 << 22) continue;
                        const int f = i8_form(gated, m, n, k);
                        if (f < 0 || f >= I8_FORMS || (gated && !I8_FORM[f].gated_channels)) return 1;
                        if (f <= I8_STREAM_32 && m > I8_STREAM_ROWS) return 2;
                        // Fewer than 2^32 threads of at most 512 a workgroup.
                        if (i8_tiles(I8_FORM[f], gated, m, n) + 8 >= 1LL << 23) return 3;
                    }
        puts("ok");
        return 0;
    }
    int gated, m, n, k;
    while (scanf("%d %d %d %d", &gated, &m, &n, &k) == 4) {
        const int f = i8_form(gated, m, n, k);
        printf("%d %d\n", f, I8_FORM[f].parts);
    }
    return 0;
}
''')
    exe = str(tmp / "forms")
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", os.path.join(ROOT, "instantcua_amd", "csrc"),
                    str(tmp / "forms.cpp"), "-o", exe], check=True)
    return exe


def test_every_size_has_a_form(exe):
    assert subprocess.run([exe, "all"], capture_output=True, text=True).stdout.strip() == "ok"


def test_the_deep_shapes_take_their_forms(exe):
    text = "".join(f"{g} {m} {n} {k}\n" for _, g, m, n, k in DEEP)
    got = [[int(x) for x in line.split()] for line in subprocess.run([exe], input=text, capture_output=True, text=True, check=True).stdout.splitlines()]
    names = [f[0] for f in FORMS]
    for (name, gated, m, n, k), (form, parts) in zip(DEEP, got):
        assert names[form] == name, (name, names[form], gated, m, n, k)
        _, groups, stages = FORMS[form]
        assert parts == groups and k // 128 // groups >= stages + 2 and k % 128
    small = ("I8_32x32", "I8_32x64", "I8_64x64_DEEP", "I8_64x64")  # not for gates
    assert {(s[0], s[1]) for s in DEEP} == {(f, g) for f in names for g in (0, 1) if not g or f not in small}
