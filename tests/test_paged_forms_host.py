"""CPU tests of the attention over paged caches with a window or shared prefixes: refusals, sizes, and the index
functions of what their kernels go through."""
import ctypes as C
import os
import subprocess

import pytest

from instantcua_amd import engine as eng
from instantcua_amd import paged
from test_paged_host import At, ROOT, cache, library  # noqa: F401


def window(**kw):
    a = dict(q=At(), out=At(), n_heads=16, q_start=At(), kv_len=At(), tables=At(), n_seqs=2, n_tokens=2, table_width=64,
             window=100, sinks=4, work=At())
    a.update(kw)
    cache().attention_window(**a)


def prefix(**kw):
    a = dict(q=At(), out=At(), n_heads=16, q_start=At(), kv_len=At(), tables=At(), n_seqs=2, n_tokens=2, table_width=64,
             group_start=At(), prefix_len=At(), n_groups=1, work=At())
    a.update(kw)
    cache().attention_prefix(**a)


@pytest.mark.parametrize("kw,match", [
    (dict(window=0), "window"), (dict(window=-1), "window"), (dict(sinks=-1), "window"), (dict(type=2), "type"),
    (dict(n_heads=12), "n_heads"), (dict(n_seqs=-1), "negative"), (dict(n_seqs=(1 << 14) + 1), "2\\^14"),
    (dict(table_width=0), "table_width"), (dict(q=None), "q and out"), (dict(tables=None), "q_start"),
    (dict(work=None), "work"), (dict(work=At(8)), "work"), (dict(work=At(nbytes=64)), "work"), (dict(scale=float("nan")), "scale"),
])
def test_window_refuses(kw, match):
    with pytest.raises(eng.EngineError, match=match):
        window(**({"window": 4000} | kw))


@pytest.mark.parametrize("kw,match", [
    (dict(n_groups=-1), "n_groups"), (dict(n_groups=65), "n_groups"), (dict(max_prefix=-1), "negative"),
    (dict(group_start=None), "group_start"), (dict(prefix_len=None), "group_start"), (dict(type=2), "type"),
    (dict(n_heads=12), "n_heads"), (dict(n_tokens=-1), "negative"), (dict(out=At(4)), "q and out"),
    (dict(work=None), "work"), (dict(work=At(nbytes=64)), "work"),
])
def test_prefix_refuses(kw, match):
    with pytest.raises(eng.EngineError, match=match):
        prefix(**kw)


def test_work_refuses():
    c = cache()
    with pytest.raises(eng.EngineError, match="window"):
        c.attention_window_work(16, 1, 1, 0)
    with pytest.raises(eng.EngineError, match="n_groups"):
        c.attention_prefix_work(16, 1, 1, 65)
    # A window's slots alone count; groups of none, or of prefixes below a step, take what the plain call takes.
    sizes = dict(max_q=1, max_kv=16384)
    assert c.attention_window_work(16, 8, 8, 1, **sizes) < c.attention_work(16, 8, 8, **sizes)
    assert c.attention_window_work(16, 8, 8, 16384, **sizes) == c.attention_work(16, 8, 8, **sizes)
    for groups, bound in ((0, 0), (3, 127)):
        assert c.attention_prefix_work(16, 8, 8, groups, bound, **sizes) == c.attention_work(16, 8, 8, **sizes)


def test_nothing_to_do_is_no_error():
    cache().attention_window(None, None, 16, None, None, None, 0, 0, 4, 10)
    cache().attention_prefix(None, None, 16, None, None, None, 0, 0, 4, None, None, 0)


def test_null_arguments():
    L, p, a, n = eng.lib(), cache(), (C.c_byte * 256)(), C.c_size_t()
    for form in ("window", "prefix"):
        assert getattr(L, f"icua_paged_attention_{form}")(p._at, C.addressof(a), None, None) != 0 and b"null" in L.icua_last_error()
        assert getattr(L, f"icua_paged_attention_{form}_work")(p._at, C.addressof(a), None, C.byref(n)) != 0


def test_structures_have_the_sizes_of_the_header(tmp_path):
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "icua.h"\nint main(void) { printf("%zu %zu", sizeof(icua_paged_window_t), '
                   'sizeof(icua_paged_prefix_t)); return 0; }\n')
    exe = str(tmp_path / "sizes")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    got = [int(x) for x in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [C.sizeof(t) for t in (paged._Window, paged._Prefix)]


def test_what_a_window_goes_through(tmp_path):
    """Every slot that some row sees is gone through once, in whole steps, and no more of them than the plan counts;
    groups of any numbers stay inside the batch."""
    src = tmp_path / "gap.cpp"
    src.write_text(r'''
#include <assert.h>
#include <limits.h>
#include <stdio.h>
#include <algorithm>
#include "icua_paged.h"
using namespace icua;
int main() {
    const int lens[] = {0, 1, 2, 31, 32, 33, 127, 128, 129, 200, 256, 300, 511, 640, 1000};
    for (int step : {32, 64, 128})
        for (int n : lens)
            for (int m : {1, 2, 16, 100, 128})
                for (int window : {1, 2, 31, 32, 33, 64, 100, 128, 129, 255, 600, 1 << 30})
                    for (int sinks : {0, 1, 31, 32, 33, 100, 128, 129, 500, 1 << 30}) {
                        const int own = n - m;  // the first row's slot, may be negative
                        const SlotGap g = window_gap(own, n, window, sinks, step);
                        assert(g.skip >= 0 && g.skip % step == 0 && g.from % step == 0);
                        const int left = std::max(0, n - g.skip);
                        if (step == 32 ? m <= 16 : true) assert(left <= window_slots(std::max(n, 1), window, sinks) || n == 0);
                        int last = -1;
                        for (int v = 0; v < left; ++v) {
                            const int s = gap_slot(g, v);
                            assert(s > last && s < n);
                            if (v % step) assert(s == last + 1);
                            for (int gone = last + 1; gone < s; ++gone) assert(gone >= sinks && gone <= own - window);
                            last = s;
                        }
                        for (int gone = last + 1; gone < n; ++gone) assert(gone >= sinks && gone <= own - window);
                    }
    assert(window_slots(1 << 30, 1 << 30, 1 << 30) == 1 << 30);
    const int odd[] = {INT_MIN, -1, 0, 1, 5, 7, 8, 9, INT_MAX};
    for (int a : odd)
        for (int b : odd)
            for (int p : {INT_MIN, -1, 0, 127, 128, 129, 1000, INT_MAX}) {
                const int start[2] = {a, b}, len[1] = {p};
                const PrefixGroup g = prefix_group(start, len, 0, 8, 900);
                assert(g.s0 >= 0 && g.s0 <= g.s1 && g.s1 <= 8 && g.n >= 0 && g.n <= 900 && g.n % 128 == 0);
                if (g.n) assert(g.s1 - g.s0 >= 2 && g.n <= p);
                if (a >= 0 && b <= 8 && (long long)b - a >= 2) assert(g.s0 == a && g.s1 == b && g.n == (p < 0 ? 0 : std::min(p, 900) / 128 * 128));
            }
    puts("ok");
}
''')
    exe = str(tmp_path / "gap")
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", "-I",
                    os.path.join(ROOT, "instantcua_amd", "csrc"), str(src), "-o", exe], check=True)
    assert subprocess.run([exe], capture_output=True, text=True, check=True).stdout.strip() == "ok"


def test_a_window_of_all_slots_takes_what_the_plain_call_takes():
    c = cache()
    for n_tokens, sizes in ((300, dict(max_q=300, max_kv=4000)), (8, dict(max_q=1, max_kv=4000))):
        plain = c.attention_work(16, 8, n_tokens, **sizes)
        for window, sinks in ((4000, 0), (3999, 1), (1, 3999), (2 ** 31 - 1, 2 ** 31 - 1), (1, 4000)):
            assert c.attention_window_work(16, 8, n_tokens, window, sinks, **sizes) == plain
