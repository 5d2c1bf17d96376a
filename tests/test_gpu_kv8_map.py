"""What the block map counts as refused, beside tests/test_gpu_kv8.py."""
import pytest
import torch

import jitllm_b200 as jl
from tests.test_gpu_kv8 import _Map, _stream

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("held,added,capacity,free,refused,lengths", [
    ((5, 5, 5), (4, 9, 0), 8, 9, 2, (9, 5, 5)),      # behind tokens that do not fit: refused without new tokens too
    ((5, 5, 5), (4, 0, 9), 8, 9, 1, (9, 5, 5)),      # in front of them: not
    ((5, 5, 5), (4, 4, 0), 8, 9, 0, (9, 9, 5)),      # the tokens just fit
    ((5, 5, 5), (4, 20, 0), 40, 0, 1, (9, 5, 5)),    # behind blocks that are not there: one that needs none is served
    ((0, 0, 0), (0, 0, 0), 0, 0, 0, (0, 0, 0))])
def test_map_counts_as_refused(dev, inplace, held, added, capacity, free, refused, lengths):
    with jl.Kv8Workspace(dev) as ws:
        m = _Map(ws, list(held), list(added), 4, 16, list(range(50, 50 + free)), 0, capacity, inplace=inplace)
        m.call.launch(_stream())
        m.check()
        torch.cuda.synchronize()
        assert int(m.result[2]) == refused and tuple(m.lengths.tolist()) == lengths
