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


@pytest.mark.parametrize("rows,token,head", [(2, 128, 128), (3, 1024 - 8, 128), (3, 128, 256), (300, 136, 40000),
                                             (1 << 20, 1 << 40, 1 << 40), (2, 1 << 62, 1 << 62)])
def test_load_refuses_strides_that_let_rows_overlap(rows, token, head):
    with pytest.raises(eng.EngineError, match="overlap"):
        cache().load(None, rows, At(), token_stride=token, head_stride=head)


@pytest.mark.parametrize("n_kv,rows,token,head", [(8, 3, 1024, 128), (8, 3, 128, 3 * 128), (8, 1, 128, 128), (1, 9, 128, 128),
                                                  (8, 300, 136, 299 * 136 + 128), (8, 2, 7 * 256 + 128, 256), (8, 5, 1 << 40, 1 << 36)])
def test_load_takes_strides_that_do_not(n_kv, rows, token, head):
    """Refused for its missing slots, which are looked at after the strides (there is no GPU here)."""
    with pytest.raises(eng.EngineError, match="slots"):
        cache(n_kv=n_kv).load(None, rows, At(), token_stride=token, head_stride=head)
