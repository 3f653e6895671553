"""moe_ffn_w4a16 where an expert has tens of routes: one, two and several passes over its weights' tiles.  Formulas and tolerances: test_gpu_w4a16."""
import pytest
import torch

from test_gpu_w4a16 import KINDS, block, check_block

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt,group,zeros", KINDS)
@pytest.mark.parametrize("m,e,top_k", [(48, 3, 2), (60, 5, 2), (72, 4, 2), (100, 4, 1), (97, 3, 3), (150, 2, 1)])
def test_tens_of_routes(m, e, top_k, fmt, group, zeros, dtype):
    check_block(*block(m + e, m, 160, 320, e, top_k, fmt, group, zeros, dtype), fmt, group)
