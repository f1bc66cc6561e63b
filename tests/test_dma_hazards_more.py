"""The check of test_dma_hazards for the other sources that hold global->LDS DMA
loads: no base register written by a VALU instruction too shortly before."""

from concurrent.futures import ThreadPoolExecutor

import pytest

from tests.test_dma_hazards import B, _device_asm, dma_hazards
from tests.test_dma_hazards import pytestmark  # noqa: F401  (skipped without hipcc)

SOURCES = ["varlen_prefill_window.hip", "paged_rows_tree.hip"]


@pytest.fixture(scope="module")
def asm_files(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("asm_more")
    with ThreadPoolExecutor(max_workers=len(SOURCES)) as ex:
        return dict(zip(SOURCES, ex.map(lambda s: _device_asm(B.CSRC / s, tmp), SOURCES)))


@pytest.mark.parametrize("src", SOURCES)
def test_no_dma_operand_hazards(asm_files, src):
    n, found = dma_hazards(asm_files[src])
    assert n > 0 and not found, f"{len(found)} DMA operand hazards in {src}:\n" + "\n".join(found[:20])
