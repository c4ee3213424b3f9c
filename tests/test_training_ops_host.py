"""Host-side behaviour of the training operators that needs no GPU: specs, refusals, and the
C entry points' argument checks (they return a status before any device work)."""
import ctypes
import math

import numpy as np
import pytest
import torch

from featgraph_b200 import _lib, module, te
from featgraph_b200 import op as ops
from featgraph_b200.build import build_library


@pytest.fixture(scope="module")
def lib():
    build_library()
    return _lib.load()


def test_specs():
    out = ops.embedding_lookup(te.placeholder((50, 12), "bfloat16"), te.placeholder((7,), "int64"),
                               scale=2, padding_idx=3, with_grad=True)
    assert out.shape == (7, 12) and out.dtype == "bfloat16" and out.kind == "embedding_lookup"
    assert out.attrs["padding_idx"] == 3 and out.attrs["scale"] == 2.0
    assert ops.schedule_embedding_lookup_cuda(out).target == "cuda"
    out = ops.softmax_cross_entropy(te.placeholder((9, 4)), te.placeholder((50, 4)),
                                    te.placeholder((9,), "int32"))
    assert out.shape == (9,) and out.attrs["vocab"] == 50 and out.attrs["ignore_index"] == -100
    out = ops.gradient_clip(te.placeholder((3, 4)), te.placeholder((5,), "float16"), max_norm=2)
    assert out.shape == (1,) and out.attrs["max_norm"] == 2.0 and not out.attrs["in_place"]


@pytest.mark.parametrize("call, error, text", [
    (lambda p: ops.embedding_lookup(p((5,)), p((3,), "int32")), ValueError, "2-D"),
    (lambda p: ops.embedding_lookup(p((5, 0)), p((3,), "int32")), ValueError, "column"),
    (lambda p: ops.embedding_lookup(p((5, 2), "float64"), p((3,), "int32")), TypeError, "dtype"),
    (lambda p: ops.embedding_lookup(p((5, 2)), p((3,), "float32")), TypeError, "dtype"),
    (lambda p: ops.embedding_lookup(p((5, 2)), p((3, 1), "int32")), ValueError, "1-D"),
    (lambda p: ops.embedding_lookup(p((5, 2)), p((3,), "int32"), padding_idx=5), ValueError, "padding"),
    (lambda p: ops.embedding_lookup(p((5, 2)), p((3,), "int32"), scale=math.nan), ValueError, "finite"),
    (lambda p: ops.softmax_cross_entropy(p((3, 2)), p((5, 3)), p((3,), "int32")), AssertionError, "mismatch"),
    (lambda p: ops.softmax_cross_entropy(p((3, 2)), p((5, 2)), p((4,), "int32")), AssertionError, "mismatch"),
    (lambda p: ops.softmax_cross_entropy(p((3, 2)), p((0, 2)), p((3,), "int32")), ValueError, "row"),
    (lambda p: ops.softmax_cross_entropy(p((3, 2)), p((5, 2), "float16"), p((3,), "int32")), TypeError, "Weight"),
    (lambda p: ops.gradient_clip(p((3,), "int32")), TypeError, "dtype"),
    (lambda p: ops.gradient_clip(p((3,)), max_norm=-1), ValueError, "negative"),
    (lambda p: ops.gradient_clip(p((3,)), max_norm=math.nan), ValueError, "negative"),
    (lambda p: ops.gradient_clip(p((3,)), norm_type=1), ValueError, "norm_type"),
    (lambda p: ops.gradient_clip(p((3,)), eps=math.inf), ValueError, "finite"),
])
def test_op_refusals(call, error, text):
    with pytest.raises(error, match=text):
        call(te.placeholder)


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU failure mode")
def test_modules_fail_loudly_without_a_gpu():
    for cls in (module.EmbeddingLookupcuda, module.SoftmaxCrossEntropycuda, module.GradientClipcuda):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            cls()


def _refused(lib, status, code, text):
    assert status == code
    assert text in lib.fg_last_error_string().decode()


def test_lookup_argument_errors(lib):
    some = ctypes.c_void_p(4096)      # never read: every call below is refused before a launch

    def call(table=some, dtype=0, ld=8, v=10, ids=some, index=0, n=5, f=8, out=some, out_ld=8,
             status=some):
        return lib.fg_embedding_lookup(table, dtype, ld, v, ids, index, n, f, 1.0, out, out_ld,
                                       status, 0, None)
    _refused(lib, call(dtype=3), 1, "dtype")
    _refused(lib, call(index=2), 1, "index_type")
    _refused(lib, call(f=0), 1, "feat_len")
    _refused(lib, call(n=-1), 1, "n_ids")
    _refused(lib, call(ld=7), 1, "pitch")
    _refused(lib, call(out_ld=7), 1, "pitch")
    _refused(lib, call(ids=None), 1, "null")
    _refused(lib, call(table=None), 1, "null")
    _refused(lib, call(n=1 << 31), 3, "2^31")
    assert call(n=0) == 0             # nothing to do, no device needed


def test_lookup_grad_argument_errors(lib):
    some = ctypes.c_void_p(4096)
    need = lib.fg_embedding_grad_workspace_bytes(5, 10, 8)
    assert need > 0 and lib.fg_embedding_grad_workspace_bytes(0, 10, 8) == 0

    def call(dy=some, ld=8, ids=some, n=5, v=10, f=8, padding=-1, grad=some, ws=some, size=need,
             dtype=0):
        return lib.fg_embedding_grad(dy, dtype, ld, ids, 0, n, v, f, 1.0, padding, 0, grad, ws,
                                     size, some, 0, None)
    _refused(lib, call(size=need - 1), 1, "workspace")
    _refused(lib, call(ws=None), 1, "workspace")
    _refused(lib, call(ws=ctypes.c_void_p(4100)), 1, "workspace")
    _refused(lib, call(padding=10), 1, "padding_id")
    _refused(lib, call(grad=None), 1, "null")
    _refused(lib, call(ld=4), 1, "pitch")
    _refused(lib, call(dtype=7), 1, "dtype")
    assert call(n=0, v=0) == 0


def test_xent_argument_errors(lib):
    some = ctypes.c_void_p(4096)
    need = lib.fg_softmax_xent_workspace_bytes(0, 5, 10, 8, 0)
    need_grad = lib.fg_softmax_xent_workspace_bytes(0, 5, 10, 8, 1)
    assert 0 < need <= need_grad

    def call(feat=some, fld=8, weight=some, wld=8, dtype=0, labels=some, index=0, n=5, v=10, d=8,
             loss=some, ws=some, size=need):
        return lib.fg_softmax_xent(feat, fld, weight, wld, dtype, labels, index, n, v, d, 1.0,
                                   -100, loss, some, ws, size, some, 0, None)
    _refused(lib, call(dtype=-1), 1, "dtype")
    _refused(lib, call(v=0), 1, "shape")
    _refused(lib, call(fld=7), 1, "shape")
    _refused(lib, call(wld=7), 1, "shape")
    _refused(lib, call(labels=None), 1, "null")
    _refused(lib, call(loss=None), 1, "null")
    _refused(lib, call(size=need - 1), 1, "workspace")
    _refused(lib, call(ws=ctypes.c_void_p(4100)), 1, "workspace")
    _refused(lib, call(n=1 << 30), 3, "2^30")
    _refused(lib, call(feat=ctypes.c_void_p(4097)), 1, "aligned")
    assert call(n=0) == 0
    for scale in (math.nan, math.inf):
        _refused(lib, lib.fg_softmax_xent(some, 8, some, 8, 0, some, 0, 5, 10, 8, scale, -100, some,
                                          some, some, need, some, 0, None), 1, "finite")

    def grad(dh=some, dw=some, size=need_grad, lse=some):
        return lib.fg_softmax_xent_grad(some, some, 8, some, 8, 0, some, 0, 5, 10, 8, 1.0, -100,
                                        lse, dh, dw, some, size, some, 0, None)
    _refused(lib, grad(dh=None, dw=None), 1, "neither")
    _refused(lib, grad(size=need_grad - 1), 1, "workspace")
    _refused(lib, grad(lse=None), 1, "null")


def test_clip_argument_errors(lib):
    some = ctypes.c_void_p(4096)
    need = lib.fg_gradient_clip_workspace_bytes(2)

    def call(sizes=(4, 4), dtypes=(0, 2), ins=(4096, 4096), n=2, max_norm=1.0, eps=1e-6, norm=some,
             size=need):
        a = (ctypes.c_void_p * 2)(*ins)
        return lib.fg_gradient_clip(a, a, (ctypes.c_int64 * 2)(*sizes), (ctypes.c_int32 * 2)(*dtypes),
                                    n, 0, max_norm, eps, norm, some, size, 0, None)
    _refused(lib, call(n=-1), 1, "n_tensors")
    _refused(lib, call(sizes=(4, -1)), 1, "tensor 1")
    _refused(lib, call(dtypes=(0, 9)), 1, "tensor 1")
    _refused(lib, call(ins=(None, 4096)), 1, "tensor 0")
    _refused(lib, call(ins=(4098, 4096)), 1, "tensor 0")
    _refused(lib, call(max_norm=-1.0), 1, "max_norm")
    _refused(lib, call(max_norm=math.nan), 1, "max_norm")
    _refused(lib, call(eps=-1.0), 1, "eps")
    _refused(lib, call(norm=None), 1, "norm_dev")
    _refused(lib, call(size=need - 1), 1, "workspace")
    _refused(lib, call(sizes=(1 << 50, 4)), 3, "chunks")
    assert lib.fg_gradient_clip(None, None, None, None, 1, 0, 1.0, 0.0, some, some, need, 0, None) == 1


def test_workspace_sizes_grow_with_the_work(lib):
    sizes = [lib.fg_embedding_grad_workspace_bytes(n, 1000, 64) for n in (1, 100, 10000, 1000000)]
    assert sizes == sorted(sizes) and sizes[0] > 0
    assert lib.fg_gradient_clip_workspace_bytes(5000) > lib.fg_gradient_clip_workspace_bytes(1) > 0
    assert np.iinfo(np.int32).max < lib.fg_embedding_grad_workspace_bytes(2000000000, 1000, 64)


def test_calls_by_words(lib):
    import struct
    words = struct.pack("=8qd5q", 4096, 0, 8, 10, 4096, 0, 0, 8, 1.0, 4096, 8, 4096, 0, 0)
    assert lib.fg_training_call(_lib.OP_LOOKUP, words, 14) == 0        # no ids: nothing to do
    _refused(lib, lib.fg_training_call(_lib.OP_LOOKUP, words, 13), 1, "takes 14")
    _refused(lib, lib.fg_training_call(9, words, 14), 1, "training_op")
    _refused(lib, lib.fg_training_call(_lib.OP_LOOKUP, None, 14), 1, "null")
    bad = struct.pack("=8qd5q", 4096, 0, 7, 10, 4096, 0, 5, 8, 1.0, 4096, 8, 4096, 0, 0)
    _refused(lib, lib.fg_training_call(_lib.OP_LOOKUP, bad, 14), 1, "pitch")
    # a number arrives as such: max_norm = -1.5 is refused by its value
    clip = struct.pack("=6qdd5q", 4096, 4096, 4096, 4096, 0, 0, -1.5, 1e-6, 4096, 4096, 1 << 20, 0, 0)
    _refused(lib, lib.fg_training_call(_lib.OP_CLIP, clip, 13), 1, "-1.5")
    for op, fields in ((_lib.OP_LOOKUP_GRAD, 17), (_lib.OP_XENT, 19), (_lib.OP_XENT_GRAD, 21)):
        _refused(lib, lib.fg_training_call(op, words, 1), 1, "takes %d" % fields)


def test_misaligned_pointers_are_refused(lib):
    some, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4098)
    odd8 = ctypes.c_void_p(4100)
    for index, ids in ((0, odd), (1, odd8)):
        _refused(lib, lib.fg_embedding_lookup(some, 0, 8, 10, ids, index, 5, 8, 1.0, some, 8, some,
                                              0, None), 1, "aligned")
        _refused(lib, lib.fg_softmax_xent(some, 8, some, 8, 0, ids, index, 5, 10, 8, 1.0, -100, some,
                                          some, some, 1 << 30, some, 0, None), 1, "aligned")
    need = lib.fg_softmax_xent_workspace_bytes(0, 5, 10, 8, 1)
    for place in range(4):
        p = [odd if k == place else some for k in range(4)]     # loss_grad, lse and the gradients
        _refused(lib, lib.fg_softmax_xent_grad(p[0], some, 8, some, 8, 0, some, 0, 5, 10, 8, 1.0,
                                               -100, p[1], p[2], p[3], some, need, some, 0, None), 1,
                 "aligned")
    _refused(lib, lib.fg_softmax_xent(some, 8, some, 8, 0, some, 0, 5, 10, 8, 1.0, -100, odd, some,
                                      some, 1 << 30, some, 0, None), 1, "aligned")
