"""Which kernel an MXFP4 product of short rows takes (no GPU needed)."""
from __future__ import annotations

import pytest


# rows, cols, batch, kernel: the K-split kernel while its 32 x 32 tiles are one round of the 256
# CUs, and where a load of 16 scales would leave an array; else tiles of 128 x 128
@pytest.mark.parametrize("rows,cols,batch,kernel", [
    (1536, 256, 128, "k32"), (1536, 256, 2000, "t128x128n"), (1536, 256, 160, "k32"),
    (1536, 256, 161, "t128x128n"), (8192, 480, 32, "k32"), (8192, 480, 33, "t128x128n"),
    (16384, 32, 16, "t128x128n"), (16384, 32, 15, "k32"), (16, 32, 8192, "k32"),
    (16, 32, 8193, "t128x128n"), (15, 32, 1 << 20, "k32"), (2000, 288, 1700, "t128x128n"),
    (5000, 64, 1, "k32")])
def test_products_of_short_rows(axc, rows, cols, batch, kernel):
    assert f"_{kernel}_" in axc.mxfp4_matmul_kernel_name(rows, cols, batch)
