"""CPU tests that attn_decode_shared refuses outputs that share memory with its tables, lengths or bounds, and only those."""
from __future__ import annotations

import attn_dispatch as D
import pytest
from test_candidates_accepts import PLEN, PTABLE, _refused, _run, shared, tmp  # noqa: F401

B, HQ, HD = 8, 8, 64
OUT_BYTES = B * HQ * HD * 2


@pytest.mark.parametrize("name,at,size", [("prefix_table", PTABLE, 2 * 8 * 4), ("table", D.TABLE, B * 8 * 4), ("prefix_len", PLEN, 2 * 4),
                                          ("kv_len", D.LEN, B * 4), ("cu_seq", D.CU, 3 * 4)])
def test_outputs_over_what_is_read(tmp, name, at, size):  # noqa: F811
    kv = D.cache(4, HD)
    up = lambda n: -(-n // 16) * 16
    _refused(tmp, f"overlaps {name}", shared(kv, B, 2, HQ, 4, HD, out=at), shared(kv, B, 2, HQ, 4, HD, out=at - OUT_BYTES + 16),
             shared(kv, B, 2, HQ, 4, HD, out=at + up(size) - 16))
    for out in (at - OUT_BYTES, at + up(size)):
        _run(tmp, shared(kv, B, 2, HQ, 4, HD, out=out), 2)


def test_tables_between_the_outputs_rows(tmp):  # noqa: F811
    """Rows of one buffer: outputs, and behind each row's end its table."""
    kv = D.cache(4, HD)
    row = HQ * HD + 64
    call = lambda table: shared(kv, B, 2, HQ, 4, HD, os=row, table=table, ts=row // 2)
    _run(tmp, call(D.OUT + HQ * HD * 2), 2)
    _refused(tmp, "overlaps table", call(D.OUT + HQ * HD * 2 - 4))


def test_tables_of_no_pages(tmp):  # noqa: F811
    kv = D.cache(4, HD)
    _run(tmp, shared(kv, B, 2, HQ, 4, HD, ppages=0, pages=0, table=D.OUT, ptable=D.OUT), 2)
