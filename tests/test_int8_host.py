"""CPU tests of the products on 8-bit integers: arguments are refused before anything is enqueued."""
import ctypes as C
import os
import subprocess

import pytest

from instantcua_amd import engine as eng
from instantcua_amd import int8

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class At:
    """A buffer that is never looked at."""

    def __init__(self, ptr, nbytes=1 << 60):
        self.ptr, self.nbytes = ptr, nbytes


G = 1 << 30  # buffers far apart


@pytest.fixture(scope="module", autouse=True)
def library():
    if not os.path.exists(eng.LIB_PATH):
        from instantcua_amd import build
        build.build()


@pytest.mark.parametrize("kw,match", [
    (dict(type=2), "type"), (dict(type=-1), "type"), (dict(n_rows=-1), "n_rows"), (dict(n_rows=(1 << 24) + 1), "n_rows"), (dict(n_cols=0), "n_cols"), (dict(x_stride=(1 << 22) + 8), "x_stride"),
    (dict(n_cols=24), "n_cols"), (dict(n_cols=-16), "n_cols"), (dict(n_cols=(1 << 17) + 16), "n_cols"),
    (dict(x_stride=2040), "x_stride"), (dict(x_stride=2052), "x_stride"), (dict(codes_stride=2032), "codes_stride"),
    (dict(codes_stride=2056), "codes_stride"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(x=None), "x and codes"), (dict(x=At(G + 8)), "x and codes"), (dict(codes=At(2 * G + 4)), "x and codes"),
    (dict(norm=At(3 * G + 4)), "norm"), (dict(scales=None), "scales"), (dict(scales=At(4 * G + 2)), "scales"),
    (dict(codes=At(G + 3 * 2048 * 4 - 16)), "overlap"), (dict(scales=At(2 * G + 16)), "overlap"),
    (dict(scales=At(3 * G + 2047 * 4)), "overlap"), (dict(codes=At(G), type=1), "overlap"),
])
def test_quantize_refuses(kw, match):
    a = dict(x=At(G), codes=At(2 * G), scales=At(4 * G), n_rows=3, n_cols=2048, norm=At(3 * G))
    a.update(kw)
    with pytest.raises(eng.EngineError, match=match):
        int8.quantize(**a)


@pytest.mark.parametrize("kw,match", [
    (dict(type=2), "type"), (dict(gated=2), "gated"), (dict(n_rows=-1), "negative"), (dict(n_out=-1), "negative"),
    (dict(n_out=(1 << 22) + 1), "2\\^22"), (dict(n_rows=1 << 20, n_out=(1 << 16) + 1), "2\\^36"),
    (dict(n_rows=(1 << 24) + 1), "2\\^24"), (dict(x_stride=(1 << 22) + 16), "x_stride"), (dict(y_stride=(1 << 22) + 1), "y_stride"), (dict(n_in=0), "n_in"),
    (dict(n_in=2040), "n_in"), (dict(n_in=(1 << 17) + 16), "n_in"), (dict(x_stride=2032), "x_stride"),
    (dict(x_stride=2056), "x_stride"), (dict(w_stride=16), "w_stride"), (dict(w_stride=2050), "w_stride"),
    (dict(add_stride=99), "add_stride"), (dict(y_stride=99), "y_stride"), (dict(gated=True, add=At(7 * G)), "gated"),
    (dict(x=None), "x and w"), (dict(w=At(3 * G + 8)), "x and w"), (dict(x_scales=None), "scales"),
    (dict(w_scales=At(4 * G + 2)), "scales"), (dict(y=None), "y must"), (dict(y=At(5 * G + 2)), "y must"),
    (dict(y=At(5 * G + 1), type=1), "y must"), (dict(add=At(7 * G + 2)), "add"), (dict(y=At(G)), "overlap"),
    (dict(y=At(3 * G)), "overlap"), (dict(y=At(2 * G)), "overlap"), (dict(y=At(4 * G + 396)), "overlap"),
    (dict(add=At(5 * G), add_stride=104), "overlap"), (dict(add=At(5 * G + 4)), "overlap"), (dict(add=At(5 * G), type=1), "overlap"),
])
def test_matmul_refuses(kw, match):
    a = dict(x=At(G), x_scales=At(2 * G), w=At(3 * G), w_scales=At(4 * G), y=At(5 * G), n_rows=3, n_out=100, n_in=2048,
             work=At(6 * G))
    a.update(kw)
    with pytest.raises(eng.EngineError, match=match):
        int8.matmul(**a)


def test_work_refuses():
    for args in ((-1, 16, 16), (1, -1, 16), (1, 1, 17)):
        with pytest.raises(eng.EngineError):
            int8.matmul_work(*args)
    assert int8.matmul_work(0, 0, 16) == 0


def test_nothing_to_do_is_no_error():
    """No rows or channels: nothing is enqueued (there is no GPU here)."""
    int8.quantize(None, None, None, 0, 2048)
    int8.matmul(None, None, None, None, None, 0, 100, 2048)
    int8.matmul(None, None, None, None, None, 5, 0, 2048)


def test_null_arguments():
    L = eng.lib()
    for call in (L.icua_i8_quantize, L.icua_i8_matmul):
        assert call(None, None) != 0 and b"null" in L.icua_last_error()
    assert L.icua_i8_matmul_work(None, None) != 0 and b"null" in L.icua_last_error()


def test_structures_have_the_sizes_of_the_header(tmp_path):
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "icua.h"\nint main(void) { printf("%zu %zu", sizeof(icua_i8_quantize_t), '
                   'sizeof(icua_i8_matmul_t)); return 0; }\n')
    exe = str(tmp_path / "sizes")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    got = [int(x) for x in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [C.sizeof(t) for t in (int8._Quantize, int8._Matmul)]
