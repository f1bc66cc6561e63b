"""The check of test_dma_hazards for attention of a chunk over the paged cache: no
base register written by a VALU instruction too shortly before a global->LDS load."""

from tests.test_dma_hazards import B, _device_asm, dma_hazards
from tests.test_dma_hazards import pytestmark  # noqa: F401  (skipped without hipcc)


def test_no_dma_operand_hazards(tmp_path):
    n, found = dma_hazards(_device_asm(B.CSRC / "paged_chunk_stream.hip", tmp_path))
    assert n > 0 and not found, f"{len(found)} DMA operand hazards:\n" + "\n".join(found[:20])
