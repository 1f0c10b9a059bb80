"""Sizes at which the C entry points' own arithmetic would leave 64 bits are refused before any launch. CPU only."""

from __future__ import annotations

import pytest


@pytest.mark.parametrize("pages,heads,tiles", [(2**60, 1, 1), (2**40, 1, 2**31 - 1), (2**50, 16383, 1), (2**62, 1, 2**20),
                                               (2**63 - 1, 16383, 2**31 - 1)])  # fmt: skip
def test_an_append_to_a_cache_beyond_64_bits(pages, heads, tiles) -> None:
    from pck.cuda import _lib

    lib = _lib.library()
    args = [16, pages, heads, tiles, 256, 16, 16, 0, 3, 256, 128, 256, 128, 16, 0, 0]
    assert lib.pck_kv4_append(_lib.KV4_APPEND.pack(*args), None) == 3 and "2^62 bytes" in lib.pck_last_error().decode()
