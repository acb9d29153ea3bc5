"""How many rows a plan's tiles have: by the rows, the adapters and the device's processors."""
import pytest

from paligemma_multimodal_system_b200 import seq_ops


@pytest.mark.parametrize("rows,adapters,processors,size", [(2368, 1, 148, 16), (2369, 1, 148, 128), (2368, 1, 147, 128), (1600, 3, 100, 16), (1601, 3, 100, 128), (2560, 40, 148, 128), (2559, 40, 148, 16),
                                                           (2559, 40, 10, 16), (1, 1, 148, 16)])
def test_tiles_go_by_the_processors(rows, adapters, processors, size):
    assert seq_ops._adapter_tile_rows(rows, adapters, processors) == size
