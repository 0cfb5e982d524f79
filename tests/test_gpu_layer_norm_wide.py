"""``gptrig.nn.layer_norm`` of rows that are not kept in registers (wider than 1024 pieces of 16 bytes, or less than a
piece), with more rows than the backward has parts for its column sums, against the same 64-bit reference and bounds as
the other widths."""

from __future__ import annotations

import pytest
import torch

from test_gpu_layer_norm import compare, inputs

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("rows", [513, 1500])
@pytest.mark.parametrize("width,dtype", [(6001, F32), (8192, F32), (9001, BF16), (5, BF16), (7, BF16), (3, F32)])
def test_column_sums_over_more_rows_than_parts(rows, width, dtype):
    print(f"layer_norm rows={rows} width={width} {dtype}", flush=True)
    for params, bias in ((F32, True), (BF16, False)):
        compare(*inputs((rows, width), dtype, params, bias, seed=rows))
