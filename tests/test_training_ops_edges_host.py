"""Edges of the training operators' host side that need no GPU."""
import ctypes
import math

import numpy as np
import pytest
import torch

from featgraph_b200 import _lib, nd, te
from featgraph_b200 import op as ops
from featgraph_b200.build import build_library


@pytest.fixture(scope="module")
def lib():
    build_library()
    return _lib.load()


def refused(lib, status, code, text):
    assert status == code and text in lib.fg_last_error_string().decode()


def test_a_bfloat16_array_comes_to_the_host_as_float32():
    x = torch.tensor([[1.5, -2.0], [3.25, 1e30]]).bfloat16()
    y = nd.NDArray(x).asnumpy()
    assert y.dtype == np.float32 and np.array_equal(y, x.float().numpy())
    assert nd.NDArray(x.half()).asnumpy().dtype == np.float16
    assert nd.NDArray(x.float()).asnumpy().dtype == np.float32


@pytest.mark.parametrize("scale", [1e39, -1e39, 2.0 ** 128 - 2.0 ** 103])
def test_a_scale_beyond_float32_is_refused(scale):
    p = te.placeholder
    with pytest.raises(ValueError, match="float32"):
        ops.embedding_lookup(p((5, 2)), p((3,), "int32"), scale=scale)
    with pytest.raises(ValueError, match="float32"):
        ops.softmax_cross_entropy(p((3, 2)), p((5, 2)), p((3,), "int32"), scale=scale)
    most = float(np.finfo(np.float32).max)
    assert ops.embedding_lookup(p((5, 2)), p((3,), "int32"), scale=most).attrs["scale"] == most


@pytest.mark.parametrize("index", [2 ** 63, -2 ** 63 - 1])
def test_an_ignore_index_beyond_64_bits_is_refused(index):
    p = te.placeholder
    with pytest.raises(ValueError, match="64 bits"):
        ops.softmax_cross_entropy(p((3, 2)), p((5, 2)), p((3,), "int32"), ignore_index=index)


def test_the_lookups_c_calls_refuse_a_scale_that_is_not_finite(lib):
    some = ctypes.c_void_p(4096)      # never read: the calls are refused before a launch
    for scale in (math.nan, math.inf, -math.inf):
        refused(lib, lib.fg_embedding_lookup(some, 0, 8, 10, some, 0, 5, 8, scale, some, 8, some, 0,
                                             None), 1, "finite")
        refused(lib, lib.fg_embedding_grad(some, 0, 8, some, 0, 5, 10, 8, scale, -1, 0, some, some,
                                           1 << 20, some, 0, None), 1, "finite")
