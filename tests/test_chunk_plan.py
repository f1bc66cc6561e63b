"""Which calls of attention of a chunk cut their items into runs, told by the workspace:
partial results where they do, else a few KB."""

import pytest

from tinyserver_amd import _lib


@pytest.mark.parametrize("seqs,blocks,cut", [
    (4, 8, False),    # short tables: not cut
    (1, 12, True),    # few items (float32's; the workspace serves every type)
    (4, 16, True),
    (40, 16, False),  # as many items as there are workgroups for
    (40, 17, True),   # longer tables: always
    (1, 17, True),
])
def test_short_tables(seqs, blocks, cut):
    n = _lib.load().tsa_paged_chunk_workspace_bytes(seqs, seqs, 1, 16, 8, 128, 2 * blocks, 16)
    assert (n > 1 << 18) == cut, n
