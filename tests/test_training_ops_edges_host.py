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


# ------------------------------------------------- results that share memory with an input --
# Addresses that are never read: every call below is refused before a launch.
def at(x):
    return ctypes.c_void_p(x)


BASE, FAR = 1 << 20, 1 << 24


def lookup(lib, table, ld, ids, out, out_ld, v=10, n=5, f=8):
    return lib.fg_embedding_lookup(at(table), 0, ld, v, at(ids), 1, n, f, 1.0, at(out), out_ld,
                                   at(FAR * 4), 99, None)


def test_a_lookup_over_its_own_input_is_refused(lib):
    table = 10 * 8 * 4
    for out in (BASE, BASE + table - 32, BASE - 5 * 32 + 32):
        refused(lib, lookup(lib, BASE, 8, FAR, out, 8), 1, "shares memory")
    refused(lib, lookup(lib, FAR, 8, BASE, BASE + 32, 8), 1, "shares memory")          # the ids
    # beside each other, also as columns of one array: the next check is the device's
    for args in ((BASE, 8, FAR, BASE + table, 8), (BASE, 8, FAR, BASE - 5 * 32, 8),
                 (BASE, 24, FAR, BASE + 32, 24), (BASE, 24, FAR, BASE + 64, 24)):
        assert lookup(lib, *args) == 2
    for args in ((BASE, 24, FAR, BASE + 28, 24), (BASE, 24, FAR, BASE + 68, 24),
                 (BASE, 24, FAR, BASE + 32, 16)):
        refused(lib, lookup(lib, *args), 1, "shares memory")


def test_a_lookup_gradient_over_its_own_input_is_refused(lib):
    def call(dy, ids, grad):
        return lib.fg_embedding_grad(at(dy), 0, 8, at(ids), 1, 5, 10, 8, 1.0, -1, 0, at(grad), at(FAR * 2),
                                     1 << 20, at(FAR * 4), 99, None)
    for dy in (BASE, BASE + 320 - 4, BASE - 160 + 4):
        refused(lib, call(dy, FAR, BASE), 1, "shares memory")
    refused(lib, call(FAR, BASE + 8, BASE), 1, "shares memory")
    assert call(BASE + 320, FAR, BASE) == 2


def test_a_cross_entropy_over_its_own_input_is_refused(lib):
    n, v, d = 5, 10, 8
    need = lib.fg_softmax_xent_workspace_bytes(0, n, v, d, 1)
    good = dict(feat=BASE, weight=BASE + 4096, labels=BASE + 8192, loss=BASE + 12288, lse=BASE + 16384,
                dl=BASE + 20480, dh=BASE + 24576, dw=BASE + 28672)

    def loss(**change):
        a = dict(good, **change)
        return lib.fg_softmax_xent(at(a["feat"]), d, at(a["weight"]), d, 0, at(a["labels"]), 1, n, v, d, 1.0,
                                   -100, at(a["loss"]), at(a["lse"]), at(FAR), need, at(FAR * 2), 99, None)

    def grad(**change):
        a = dict(good, **change)
        return lib.fg_softmax_xent_grad(at(a["dl"]), at(a["feat"]), d, at(a["weight"]), d, 0, at(a["labels"]),
                                        1, n, v, d, 1.0, -100, at(a["lse"]), at(a["dh"]), at(a["dw"]), at(FAR),
                                        need, at(FAR * 2), 99, None)
    assert loss() == 2 and grad() == 2
    for out in ("loss", "lse"):
        for inp in ("feat", "weight", "labels"):
            refused(lib, loss(**{out: good[inp]}), 1, "shares memory")
    refused(lib, loss(loss=good["lse"]), 1, "shares memory")
    for out in ("dh", "dw"):
        for inp in ("feat", "weight", "labels", "dl", "lse"):
            refused(lib, grad(**{out: good[inp] - 4 * (out == "dw")}), 1, "shares memory")
    refused(lib, grad(dh=good["dw"]), 1, "shares memory")
    assert grad(dl=good["lse"]) == 2                     # inputs may be one array
    # without samples the table's gradient is still written: with zeros
    refused(lib, lib.fg_softmax_xent_grad(None, None, d, at(BASE), d, 0, None, 1, 0, v, d, 1.0, -100, None,
                                          None, at(BASE + 32), None, 0, None, 99, None), 1, "shares memory")


@pytest.mark.parametrize("count", [3, 700])              # more than a launch's list too
def test_clipping_over_another_tensor_is_refused(lib, count):
    need = lib.fg_gradient_clip_workspace_bytes(count)

    def call(ins, outs, sizes, norm=FAR * 4):
        p = ctypes.c_void_p * count
        return lib.fg_gradient_clip(p(*ins), p(*outs), (ctypes.c_int64 * count)(*sizes),
                                    (ctypes.c_int32 * count)(), count, 0, 1.0, 0.0, at(norm), at(FAR * 2),
                                    need, 99, None)
    ins = [BASE + 400 * k for k in range(count)]
    outs = [FAR + 400 * k for k in range(count)]
    sizes = [100] * count
    assert call(ins, outs, sizes) == 2 and call(ins, ins, sizes) == 2
    swapped = outs[:]
    swapped[0], swapped[1] = swapped[1], swapped[0]
    refused(lib, call(outs, swapped, sizes), 1, "shares memory")       # each the other's input
    refused(lib, call(ins, [outs[0]] * 2 + outs[2:], sizes), 1, "shares memory")
    refused(lib, call(ins, [ins[0] + 4] + outs[1:], sizes), 1, "shares memory")   # its own in part
    refused(lib, call([ins[1]] + ins[1:], [outs[0]] + ins[1:], sizes), 1, "shares memory")
    assert call([ins[0]] * count, outs, sizes) == 2                    # inputs may be one array
    for norm in (ins[2], ins[2] + 396, outs[1], outs[count - 1] + 396):
        refused(lib, call(ins, outs, sizes, norm), 1, "shares memory")
    assert call(ins, outs, sizes, outs[count - 1] + 400) == 2 and call(ins, outs, sizes, BASE - 4) == 2
    assert call(ins, [outs[0]] * 2 + outs[2:], [100, 0] + sizes[2:]) == 2    # empty: nowhere


@pytest.mark.parametrize("n", [100, 9000])               # both forms of the gradient
def test_a_gradient_of_rows_too_long_is_refused_before_any_launch(lib, n):
    f = 1 << 24
    big = 1 << 44                                        # apart by more than the arrays' size
    args = (at(big), 0, f, at(2 * big), 1, n, 10, f, 1.0, -1, 0, at(3 * big), at(4 * big), 1 << 44, at(FAR),
            99, None)
    refused(lib, lib.fg_embedding_grad(*args), 3, "too large")


@pytest.mark.parametrize("with_grad", [0, 1])
def test_a_table_in_place_needs_no_room_but_one_that_is_packed_does(lib, with_grad):
    n, v, d = 5, 1000, 64
    for dtype in (0, 1, 2):
        full = lib.fg_softmax_xent_workspace_bytes(dtype, n, v, d, with_grad)
        less = lib.fg_softmax_xent_workspace_bytes(dtype, n, v, d, with_grad + _lib.XENT_TABLE_IN_PLACE)
        assert less == full if dtype == 0 else full - less >= v * d * 2
        if with_grad:                                     # any other value but 0 asks for the gradients
            for other in (2, 3, 255, -1 - _lib.XENT_TABLE_IN_PLACE):
                assert lib.fg_softmax_xent_workspace_bytes(dtype, n, v, d, other) == full
    full = lib.fg_softmax_xent_workspace_bytes(1, n, v, d, with_grad)
    less = lib.fg_softmax_xent_workspace_bytes(1, n, v, d, with_grad + _lib.XENT_TABLE_IN_PLACE)

    def call(weight, ld, size):
        if with_grad:
            return lib.fg_softmax_xent_grad(at(BASE), at(BASE + 64), d, at(weight), ld, 1, at(BASE + 8192), 0,
                                            n, v, d, 1.0, -100, at(BASE + 12288), at(FAR * 5), at(FAR * 6),
                                            at(FAR * 3), size, at(FAR * 4), 99, None)
        return lib.fg_softmax_xent(at(BASE + 64), d, at(weight), ld, 1, at(BASE + 8192), 0, n, v, d, 1.0,
                                   -100, at(BASE + 12288), at(BASE + 16384), at(FAR * 3), size, at(FAR * 4),
                                   99, None)
    assert call(FAR, 64, less) == 2 and call(FAR, 72, less) == 2 and call(FAR + 2, 64, full) == 2
    refused(lib, call(FAR, 64, less - 1), 1, "workspace")
    for weight, ld in ((FAR + 2, 64), (FAR + 8, 64), (FAR, 65), (FAR, 68)):
        refused(lib, call(weight, ld, less), 1, "workspace")
        refused(lib, call(weight, ld, full - 1), 1, "workspace")


# ------------------------------------------------------------------------ the command --
@pytest.mark.parametrize("kernel", ["lookup", "lookup-grad", "cross-entropy", "clip", "train-step"])
def test_the_command_refuses_an_empty_batch_and_a_graph_without_edges(kernel):
    import types
    from featgraph_b200 import bench_cli
    for samples in ("0", "-3"):
        with pytest.raises(SystemExit, match="at least 1"):
            bench_cli.main(["--kernel", kernel, "--samples", samples])
    args = types.SimpleNamespace(kernel=kernel, dtype="float32", samples=3, feat_len="8")
    empty = types.SimpleNamespace(nnz=0, n_rows=5, n_cols=5, indices=torch.empty(0, dtype=torch.int32))
    with pytest.raises(SystemExit, match="there are none"):
        bench_cli._run_training(args, empty, "empty", torch.device("cpu"))
