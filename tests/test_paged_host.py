"""CPU tests of the paged-cache calls: arguments are refused before anything is enqueued, and the
functions that every index from device memory passes through stay inside the buffers."""
import ctypes as C
import os
import subprocess

import pytest

from instantcua_amd import engine as eng
from instantcua_amd import paged
from instantcua_amd.modelfile import WeightFormat

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class At:
    """A buffer that is never looked at."""

    def __init__(self, ptr=1 << 20, nbytes=1 << 60):
        self.ptr, self.nbytes = ptr, nbytes


@pytest.fixture(scope="module", autouse=True)
def library():
    if not os.path.exists(eng.LIB_PATH):
        from instantcua_amd import build
        build.build()


def cache(fmt=WeightFormat.F16, n_kv=8, page=64, pages=100, **kw):
    b = dict(k=At(), v=At(), k_scales=At(), v_scales=At())
    b.update(kw)
    return paged.PagedCache(fmt, n_kv, page, pages, **b)


@pytest.mark.parametrize("kw,match", [
    (dict(page=24), "page_slots"), (dict(n_kv=1025), "n_kv"), (dict(page=1 << 20, pages=1 << 10), "2\\^31"),
    (dict(k=At(8)), "aligned"), (dict(v=At(None)), "must be set"), (dict(fmt=WeightFormat.Q8, k_scales=At(4)), "scales"),
])
def test_pools_are_checked(kw, match):
    c = cache(**kw)
    for call in (lambda: c.store(At(), 1, At(), n_heads=16, q=At()), lambda: c.load(At(), 1, At(), At()),
                 lambda: c.attention(At(), At(), 16 * (c.n_kv // 8), At(), At(), At(), 1, 1, 4, work=At())):
        with pytest.raises(eng.EngineError, match=match):
            call()


def test_pools_are_checked_by_the_wrapper():
    for args in ((WeightFormat.Q4, 8, 64, 4), (WeightFormat.F16, 0, 64, 4), (WeightFormat.F16, 8, 64, -1)):
        with pytest.raises(eng.EngineError):
            paged.PagedCache(*args, At(), At())
    with pytest.raises(eng.EngineError, match="bytes"):
        paged.PagedCache(WeightFormat.F16, 8, 64, 4, At(nbytes=8 * 64 * 4 * 256 - 1), At())
    c = cache()
    assert list(c.slots([7, 2], 62, 4)) == [7 * 64 + 62, 7 * 64 + 63, 2 * 64, 2 * 64 + 1]
    assert c.slots([7], 0, 0).size == 0
    for args in (([7, 2], 100, 29), ([7, 2], -1, 2), ([100], 0, 1), ([-1], 0, 1)):
        with pytest.raises(eng.EngineError, match="outside"):
            c.slots(*args)


@pytest.mark.parametrize("kw,match", [
    (dict(type=2), "type"), (dict(q_type=-1), "type"), (dict(n_tokens=-1), "negative"), (dict(n_heads=-1), "n_heads"),
    (dict(n_tokens=(1 << 22) + 1), "2\\^27"), (dict(qkv_stride=32 * 128 - 8), "qkv_stride"), (dict(qkv_stride=32 * 128 + 4), "qkv_stride"),
    (dict(q_stride=16 * 128 - 8), "q_stride"), (dict(qkv=At(4)), "qkv"), (dict(qkv=None), "qkv"), (dict(q=None), "q must"),
    (dict(q_norm=At(4)), "q_norm"), (dict(k_norm=At(4)), "k_norm"), (dict(slots=None), "slots"),
    (dict(rot_dim=12), "rot_dim"), (dict(rot_dim=136), "rot_dim"), (dict(rot_dim=-8), "rot_dim"),
    (dict(rope=None, rot_dim=64), "table"), (dict(rope=At(8)), "table"), (dict(pos=None), "positions"),
    (dict(rope_rows=0), "empty"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
])
def test_store_refuses(kw, match):
    a = dict(qkv=At(), n_tokens=3, slots=At(), n_heads=16, q=At(), q_norm=At(), k_norm=At(), rope=At(), rope_rows=9,
             pos=At())
    a.update(kw)
    with pytest.raises(eng.EngineError, match=match):
        cache().store(**a)


@pytest.mark.parametrize("kw,match", [
    (dict(type=2), "type"), (dict(n_heads=12), "n_heads"), (dict(n_heads=0), "n_heads"), (dict(n_heads=136), "n_heads"),
    (dict(n_seqs=-1), "negative"), (dict(n_tokens=-1), "negative"), (dict(max_q=-1), "negative"),
    (dict(max_kv=-1), "negative"), (dict(n_seqs=(1 << 18) + 1), "2\\^21"), (dict(n_tokens=(1 << 22) + 1), "2\\^26"),
    (dict(n_seqs=1 << 18, table_width=1 << 13, max_kv=0), "2\\^36"), (dict(table_width=0), "table_width"), (dict(table_width=1 << 24), "table_width"), (dict(q_stride=8), "q_stride"),
    (dict(out_stride=16 * 128 + 4), "out_stride"), (dict(scale=float("inf")), "scale"), (dict(q=At(2)), "q and out"),
    (dict(out=None), "q and out"), (dict(q_start=None), "q_start"), (dict(kv_len=None), "q_start"),
    (dict(tables=None), "q_start"), (dict(work=None), "work"), (dict(work=At(nbytes=64)), "work"),
    (dict(work=At(8)), "work"),
])
def test_attention_refuses(kw, match):
    a = dict(q=At(), out=At(), n_heads=16, q_start=At(), kv_len=At(), tables=At(), n_seqs=2, n_tokens=2, table_width=64,
             work=At())
    a.update(kw)
    with pytest.raises(eng.EngineError, match=match):
        cache().attention(**a)


@pytest.mark.parametrize("kw,match", [
    (dict(type=3), "type"), (dict(n_rows=-1), "negative"), (dict(n_rows=(1 << 24) + 1), "2\\^27"), (dict(k=At(4)), "aligned"), (dict(slots=None), "slots"),
    (dict(token_stride=8, head_stride=128), "strides"), (dict(token_stride=128), "strides"),
    (dict(token_stride=132, head_stride=1024), "strides"),
])
def test_load_refuses(kw, match):
    a = dict(slots=At(), n_rows=3, k=At(), v=At())
    a.update(kw)
    with pytest.raises(eng.EngineError, match=match):
        cache().load(**a)


def test_nothing_to_do_is_no_error():
    """No tokens, sequences or rows: nothing is enqueued (there is no GPU here)."""
    cache().store(None, 0, None, n_heads=16)
    cache().attention(None, None, 16, None, None, None, 0, 0, 4)
    cache().load(None, 0)
    cache().load(At(), 5)


def test_null_arguments():
    p = cache()
    for call in (eng.lib().icua_paged_store, eng.lib().icua_paged_load, eng.lib().icua_paged_attention):
        assert call(p._at, None, None) != 0 and b"null" in eng.lib().icua_last_error()
        a = (C.c_byte * 256)()
        assert call(None, C.addressof(a), None) != 0 and b"null" in eng.lib().icua_last_error()
    assert eng.lib().icua_paged_attention_work(p._at, None, None) != 0


def test_structures_have_the_sizes_of_the_header(tmp_path):
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "icua.h"\nint main(void) { printf("%zu %zu %zu %zu", sizeof(icua_pages_t), '
                   'sizeof(icua_paged_store_t), sizeof(icua_paged_attention_t), sizeof(icua_paged_load_t)); return 0; }\n')
    exe = str(tmp_path / "sizes")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    got = [int(x) for x in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [C.sizeof(t) for t in (paged._Pages, paged._Store, paged._Attention, paged._Load)]


def test_indexes_from_device_memory_stay_inside(tmp_path):
    """The kernels' own index functions, over numbers at and beyond every border."""
    src = tmp_path / "index.cpp"
    src.write_text(r'''
#include <assert.h>
#include <limits.h>
#include <stdio.h>
#include <vector>
#include "icua_paged.h"
using namespace icua;
int main() {
    const int odd[] = {INT_MIN, INT_MIN + 1, -65, -1, 0, 1, 15, 16, 63, 64, 65, 1000, 1 << 20, INT_MAX - 1, INT_MAX};
    const PageMap maps[] = {{1, 1, 16}, {7, 8, 64}, {5, 3, 48}, {1, 8, 4224}, {32767, 1024, 32}, {1, 1, 2147483632}};
    for (const PageMap& m : maps) {
        const long long rows = (long long)m.n_pages * m.n_kv * m.page_slots, slots = (long long)m.n_pages * m.page_slots;
        for (int s : odd) {
            const int r = pool_slot_row(m, s);
            const bool in = s >= 0 && s < slots;
            assert(in == (r >= 0));
            if (in) {
                const long long page = s / m.page_slots, last = r + (long long)(m.n_kv - 1) * m.page_slots;
                assert(r == page * m.n_kv * m.page_slots + s % m.page_slots && last < rows);
            }
            // The same number as a page of a table.
            const int32_t table[2] = {s, 0};
            for (int at : {0, m.page_slots - 1, m.page_slots, INT_MAX})
                for (int width : {1, 2}) {
                    const int q = seq_slot_row(m, table, width, at);
                    const long long i = at / m.page_slots;
                    const bool there = i < width && table[i < 2 ? i : 0] >= 0 && table[i < 2 ? i : 0] < m.n_pages;
                    assert(there == (q >= 0));
                    if (there) assert(q + (long long)(m.n_kv - 1) * m.page_slots < rows && q % m.page_slots == at % m.page_slots);
                }
        }
    }
    for (int a : odd)
        for (int b : odd)
            for (int n : odd) {
                const int32_t start[2] = {a, b}, len[1] = {n};
                const SeqSpan s = seq_span(start, len, 0, 100, 640);
                assert(s.t0 >= 0 && s.n_q >= 0 && s.t0 + s.n_q <= 100 && s.n_kv >= 0 && s.n_kv <= 640);
                if (a >= 0 && a <= b && b <= 100) assert(s.t0 == a && s.n_q == b - a);
                if (n >= 0 && n <= 640) assert(s.n_kv == n);
            }
    puts("ok");
}
''')
    exe = str(tmp_path / "index")
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", "-I",
                    os.path.join(ROOT, "instantcua_amd", "csrc"), str(src), "-o", exe], check=True)
    assert subprocess.run([exe], capture_output=True, text=True, check=True).stdout.strip() == "ok"
