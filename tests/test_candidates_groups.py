"""CPU tests of how much of the workspace a step of many small groups takes: what would be launched is recorded, nothing
runs."""
from __future__ import annotations

import attn_dispatch as D
import pytest
from test_candidates_accepts import _refused, _run, shared, tmp  # noqa: F401


@pytest.mark.parametrize("B,G,hq,hkv,hd", [
    (4096, 4096, 8, 8, 128), (512, 512, 32, 32, 256), (2048, 2048, 32, 4, 256), (2048, 700, 64, 1, 128), (4096, 512, 32, 32, 128),
    (1 << 16, 1 << 16, 4, 4, 64), (1 << 16, 1, 4, 1, 64), (1 << 16, 1 << 16, 1, 1, 256), (16, 16, 4096, 4096, 256),
    (1, 1, 32768, 32768, 256), (3, 1 << 16, 4096, 4096, 256), (1024, 1024, 64, 2, 256)])
@pytest.mark.parametrize("i8", [False, True])
def test_up_to_2_24_query_values(tmp, B, G, hq, hkv, hd, i8):  # noqa: F811
    """Whatever groups the sequences are in, in units that do not depend on how many rows a tile could hold."""
    assert B * hq * hd <= 1 << 24
    kv = D.cache(hkv, hd, pages=4096, page=16, dtype=D.I8 if i8 else D.BF16)
    got = _run(tmp, shared(kv, B, G, hq, hkv, hd), 2)
    assert all(0 < g < 1 << 24 for _, g in got), got


def test_past_what_the_workspace_holds(tmp):  # noqa: F811
    kv = lambda h, d: D.cache(h, d, pages=4096, page=16)
    _refused(tmp, "workspace holds", shared(kv(8, 128), 1 << 15, 1 << 15, 8, 8, 128), shared(kv(1, 64), 1 << 14, 1, 64, 1, 64),
             shared(kv(16, 256), 1 << 13, 3, 16, 16, 256))
    # two sequences of one head, in groups of their own: sums of 264 bytes, two of each sequence, and three for a cut (the
    # two may be in one group: two rows of a prefix's part, or one of own keys')
    few = 5 << 20
    for n, ok in ((few + 7 * 264, True), (few + 7 * 264 - 1, False)):
        call = shared(kv(1, 64), 2, 2, 1, 1, 64, nws=n)
        _run(tmp, call, 2) if ok else _refused(tmp, "workspace holds", call)
