"""Host logic of the patch's chunk steps, on the CPU: the checks before any launch, and
the table mirror's rows, which a chunk step's kernel reads in place of a gathered
table."""

import pytest
import torch

from tinyserver_amd.inference_context import InferenceContext
from tinyserver_amd.patches import device_metadata
from tinyserver_amd.patches.block_tables import BlockTableMirror

CPU = torch.device("cpu")


def _chunk(*seqs):
    return InferenceContext("chunk", [{"context_len": c, "num_tokens": n, "block_table": t} for c, n, t in seqs])


@pytest.mark.parametrize("seqs,tokens,page,match", [
    ([(0, 3, [0])], 4, 16, "sum to 3"),
    ([(5, 0, [0]), (0, 2, [1])], 2, 16, "positive"),
    ([(-1, 2, [1])], 2, 16, "negative"),
    ([(16, 1, [4])], 1, 16, "does not hold"),
    ([(3, 2, [4, 5]), (0, 9, [1, 2])], 11, 4, "does not hold"),
    ([(0, 3, [0])], 3, None, "block_size"),
])
def test_refusals(seqs, tokens, page, match):
    with pytest.raises(ValueError, match=match):
        device_metadata(_chunk(*seqs), torch.zeros(1, tokens, dtype=torch.long), tokens, CPU, page)


def test_a_context_length_that_is_missing():
    ctx = InferenceContext("chunk", [{"num_tokens": 1, "block_table": [0]}])
    with pytest.raises(KeyError, match="context_len"):
        device_metadata(ctx, torch.zeros(1, 1, dtype=torch.long), 1, CPU, 16)


def test_no_cpu_path():
    with pytest.raises((RuntimeError, ValueError), match="(?i)gpu|cuda|device"):
        device_metadata(_chunk((3, 2, [4])), torch.tensor([[3, 4]]), 2, CPU, 16)


def test_rows_of_the_mirror():
    mirror = BlockTableMirror(CPU, rows=4, width=2)
    a, b, c = [7, 8], [9], [1, 2, 3]
    for lists in ([a, b], [b, c, a], [c], [a, c]):
        rows, extra, width = mirror.sync(lists, [5, 6])
        assert rows.dtype == extra.dtype == torch.int32 and extra.tolist() == [5, 6]
        assert width == max(len(x) for x in lists)
        for r, x in zip(rows.tolist(), lists):
            assert mirror.table[r, : len(x)].tolist() == x
        table, _ = mirror.gather(lists)
        assert table.tolist() == [x + [0] * (width - len(x)) for x in lists]
        a.append(10 + len(a))
