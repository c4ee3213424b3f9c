"""Edges of the training operators' host side that need no GPU."""
import numpy as np
import torch

from featgraph_b200 import nd


def test_a_bfloat16_array_comes_to_the_host_as_float32():
    x = torch.tensor([[1.5, -2.0], [3.25, 1e30]]).bfloat16()
    y = nd.NDArray(x).asnumpy()
    assert y.dtype == np.float32 and np.array_equal(y, x.float().numpy())
    assert nd.NDArray(x.half()).asnumpy().dtype == np.float16
    assert nd.NDArray(x.float()).asnumpy().dtype == np.float32
