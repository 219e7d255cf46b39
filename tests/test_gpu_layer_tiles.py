"""The layers' products in every tile that the host chooses among, against 64 bits: several steps of depth, parts, workgroups that go on from tile
to tile, edges.  That the sizes take these tiles is tested without a GPU."""
import pytest
import torch

from layer_tiles import FLOATS, TILES
from test_gpu_checkpoint_layers import check_linear

pytestmark = pytest.mark.gpu


CASES = [(t, dtype) for t in TILES for dtype in ((torch.float32,) if t[0] == FLOATS else (torch.float16, torch.bfloat16))]


@pytest.mark.parametrize("case,dtype", CASES, ids=lambda v: str(v).replace("torch.", "").replace(" ", ""))
def test_products_in_every_tile(case, dtype):
    what, sizes = case[1], case[5]
    acts = (None, "gelu") if what == "forward" else ("gelu", "silu") if what in ("codes", "finished") else (None, "gelu_tanh")
    for n, act in enumerate(acts):
        check_linear(*sizes, dtype, act, n == 0, n == 1)
