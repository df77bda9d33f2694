"""CPU tests of paged-cache calls that are refused since they would run for very long or give outputs that depend
on the order of writes, and of the wrapper's sizes."""
import pytest

from instantcua_amd import engine as eng
from test_paged_host import At, cache, library  # noqa: F401 (library: builds it if need be)


def attention(n_seqs, **kw):
    cache().attention(At(), At(), 16, At(), At(), At(), n_seqs, 2, 64, work=At(), **kw)


def test_more_sequences_than_a_call_takes():
    with pytest.raises(eng.EngineError, match="2\\^14"):
        attention((1 << 14) + 1, max_kv=128)
    with pytest.raises(eng.EngineError, match="2\\^14"):
        cache().attention_work(16, (1 << 14) + 1, 2, max_kv=128)
    assert cache().attention_work(16, 1 << 14, 2, max_kv=256) > 0
