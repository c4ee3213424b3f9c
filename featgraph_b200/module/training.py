"""Module classes of the training operators, with the interface of the SpMM and SDDMM modules
(``build`` fixes the shapes and allocates the outputs, ``run`` launches and returns the same
arrays every call): the vertex embedding lookup that feeds an SpMM, the softmax cross entropy
that reads its output, and the gradient clip before the optimiser.  The reference has no
counterpart (python/featgraph/module/__init__.py:1-2).

A module's outputs and workspace are shared state: one call at a time per module.  A call on
another stream than the module's last one waits for that one first; while a stream is being
captured nothing is waited for, so two graphs that hold calls of one module must not be
replayed side by side.
"""
import ctypes
import math

import torch

from .. import _lib
from ..op import training as ops
from ..runtime import NDArray, gpu, zeros
from .base import time_launches

_TORCH_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16,
                 "int32": torch.int32, "int64": torch.int64}


class _TrainingOp(object):
    """What the three modules share: device, workspace, status word, stream hand-over."""
    _compute_func = None
    _schedule_func = None

    def __init__(self, device_id=0):
        if not torch.cuda.is_available():
            raise RuntimeError("%s needs a CUDA device; there is no CPU fallback"
                               % type(self).__name__)
        _lib.load()
        self._target = "cuda"
        self._ctx = gpu(int(device_id))
        self._device = self._ctx.torch_device
        self._spec = None
        self.out_tvm = None

    def _specialise(self, input_placeholders, compute_args, schedule_args):
        out = type(self)._compute_func(*input_placeholders, **compute_args)
        return out, type(self)._schedule_func(out, **schedule_args)

    def build(self, input_placeholders, compute_args, schedule_args):
        """Fix the static shapes; allocate the outputs and the workspace."""
        out, _ = self._specialise(input_placeholders, compute_args, schedule_args)
        self._spec = None
        self._owned = []
        self._status = self._own(torch.zeros(1, dtype=torch.int32, device=self._device))
        self._allocate(out)
        size = max(self._workspace_bytes(out), 16)
        self._workspace = self._own(torch.empty(size, dtype=torch.uint8, device=self._device))
        self._workspace_size = size
        self._last_stream = torch.cuda.current_stream(self._device)
        self._spec = out

    def _own(self, tensor):
        self._owned.append(tensor)
        return tensor

    def _own_zeros(self, shape, dtype):
        a = zeros(shape, dtype, self._ctx)
        self._own(a.torch)
        return a

    def lower_to_ir(self, input_placeholders, compute_args, schedule_args):
        """One line on what ``build`` would set up with the same arguments."""
        out, sched = self._specialise(input_placeholders, compute_args, schedule_args)
        return "%r: workspace %d bytes | hints: %r" % (out, self._workspace_bytes(out), sched.hints)

    def _stream(self):
        """The current stream's handle, ordered behind the module's last call."""
        stream = torch.cuda.current_stream(self._device)
        if stream != self._last_stream:
            if not torch.cuda.is_current_stream_capturing():
                stream.wait_stream(self._last_stream)
                for t in self._owned:
                    t.record_stream(stream)
                self._last_stream = stream
        return ctypes.c_void_p(stream.cuda_stream)

    def _need(self, count, inputs, what):
        if self._spec is None:
            raise RuntimeError("build() must be called before %s" % what)
        if len(inputs) != count:
            raise ValueError("%s takes exactly %d input arrays, got %d" % (what, count, len(inputs)))

    def _tensor(self, x, shape, dtype, what, rows=False):
        """Check one input against its placeholder; ``rows``: a 2-D array whose rows may lie
        apart (each row itself contiguous)."""
        t = x.torch if isinstance(x, NDArray) else x
        if not isinstance(t, torch.Tensor):
            raise TypeError("%s: expected an NDArray or a torch.Tensor, got %r" % (what, type(x)))
        if t.dtype != _TORCH_DTYPES[dtype]:
            raise TypeError("%s: dtype %s does not match the placeholder's %s" % (what, t.dtype,
                                                                                 dtype))
        if tuple(t.shape) != shape:
            raise ValueError("%s: shape %r does not match the placeholder's %r"
                             % (what, tuple(t.shape), shape))
        if t.device != self._device:
            raise ValueError("%s: array lives on %s, the module on %s" % (what, t.device,
                                                                          self._device))
        if not t.is_contiguous():
            if not rows:
                raise ValueError("%s: array must be C-contiguous" % what)
            if (t.stride(1) != 1 and shape[1] > 1) or (t.stride(0) < shape[1] and shape[0] > 1):
                raise ValueError("%s: every row must be contiguous and the rows apart, got "
                                 "strides %r" % (what, t.stride()))
        return t

    @staticmethod
    def _pitch(t):
        return max(t.stride(0), t.shape[1]) if t.shape[0] > 1 else t.shape[1]

    def device_status(self):
        """Synchronise and return the status word: 0 when every id and label so far was in
        range; raises FeatGraphError otherwise (once: the word is then cleared)."""
        if self._spec is None:
            return 0
        torch.cuda.synchronize(self._device)
        code = int(self._status.item())
        if code:
            self._status.zero_()
            torch.cuda.synchronize(self._device)
            raise _lib.FeatGraphError(code, "%s %s" % (
                type(self).__name__, "met an index out of range" if code == 1
                else "gave up a bounded wait: its results are not to be used"))
        return 0

    @property
    def ctx(self):
        return self._ctx

    @property
    def target(self):
        return self._target


class EmbeddingLookupcuda(_TrainingOp):
    """Vertex embedding lookup with scaling, and its gradient.

        m = EmbeddingLookupcuda()
        m.build([Table (V, F), Ids (n,)], {'scale': s, 'padding_idx': p, 'with_grad': True}, {})
        out = m.run([table, ids])                  # (n, F): s * table[ids]
        grad = m.run_grad([out_grad, ids])         # (V, F): the table's gradient

    Its gradient sorts the ids and sums the rows of each vertex in fp32 in an order that the
    ids alone fix.  An id out of range gives a row of NaN, adds to no gradient and is
    reported by ``device_status``."""
    _compute_func = staticmethod(ops.embedding_lookup)
    _schedule_func = staticmethod(ops.schedule_embedding_lookup_cuda)

    def _allocate(self, out):
        table, ids = out.inputs
        self.out_tvm = self._own_zeros(out.shape, out.dtype)
        self.grad_tvm = None
        if out.attrs["with_grad"]:
            self.grad_tvm = self._own_zeros(table.shape, table.dtype)
        self._codes = (_lib.DTYPES.index(table.dtype), _lib.INDEX_TYPES.index(ids.dtype))

    def _workspace_bytes(self, out):
        if not out.attrs["with_grad"]:
            return 0
        return int(_lib.load().fg_embedding_grad_workspace_bytes(
            out.shape[0], out.attrs["num_vertices"], out.attrs["feat_len"]))

    def _launch(self, table, ids):
        a = self._spec.attrs
        _lib.check(_lib.load().fg_embedding_lookup(
            table.data_ptr(), self._codes[0], self._pitch(table), a["num_vertices"],
            ids.data_ptr(), self._codes[1], self._spec.shape[0], a["feat_len"], a["scale"],
            self.out_tvm.torch.data_ptr(), a["feat_len"], self._status.data_ptr(),
            self._ctx.device_id, self._stream()))

    def _checked_inputs(self, inputs):
        self._need(2, inputs, "run()")
        tp, ip = self._spec.inputs
        return (self._tensor(inputs[0], tp.shape, tp.dtype, "Table", rows=True),
                self._tensor(inputs[1], ip.shape, ip.dtype, "Ids"))

    def run(self, input_tvm_ndarrays):
        """[Table, Ids] -> ``self.out_tvm``, the same array every call."""
        self._launch(*self._checked_inputs(input_tvm_ndarrays))
        return self.out_tvm

    def measure_average_time(self, input_tvm_ndarrays, num_runs):
        """Mean seconds of the lookup over ``num_runs`` launches."""
        table, ids = self._checked_inputs(input_tvm_ndarrays)
        return time_launches(self._ctx, lambda: self._launch(table, ids), num_runs)

    def run_grad(self, input_tvm_ndarrays, accumulate_into=None):
        """[OutGrad (n, F), Ids] -> the table's gradient (V, F): ``self.grad_tvm``, the same
        array every call, every element overwritten.  ``accumulate_into``: a contiguous (V, F)
        array of the table's type (say, the gradient that a loss with tied weights left) that
        the sums are added onto instead; it is returned."""
        self._need(2, input_tvm_ndarrays, "run_grad()")
        a = self._spec.attrs
        if not a["with_grad"]:
            raise RuntimeError("run_grad() needs build(..., {'with_grad': True}, ...)")
        tp, ip = self._spec.inputs
        dy = self._tensor(input_tvm_ndarrays[0], self._spec.shape, tp.dtype, "OutGrad", rows=True)
        ids = self._tensor(input_tvm_ndarrays[1], ip.shape, ip.dtype, "Ids")
        if accumulate_into is None:
            result, grad = self.grad_tvm, self.grad_tvm.torch
        else:
            result = accumulate_into
            grad = self._tensor(accumulate_into, tp.shape, tp.dtype, "accumulate_into")
        padding = -1 if a["padding_idx"] is None else a["padding_idx"]
        _lib.check(_lib.load().fg_embedding_grad(
            dy.data_ptr(), self._codes[0], self._pitch(dy), ids.data_ptr(), self._codes[1],
            self._spec.shape[0], a["num_vertices"], a["feat_len"], a["scale"], padding,
            accumulate_into is not None, grad.data_ptr(), self._workspace.data_ptr(),
            self._workspace_size, self._status.data_ptr(), self._ctx.device_id, self._stream()))
        return result


class SoftmaxCrossEntropycuda(_TrainingOp):
    """Softmax cross entropy over all vertices (or classes) without keeping the logits.

        m = SoftmaxCrossEntropycuda()
        m.build([Feat (n, F), Weight (V, F), Labels (n,)],
                {'scale': s, 'ignore_index': -100, 'with_grad': True}, {})
        loss, lse = m.run([feat, weight, labels])                        # both (n,) float32
        feat_grad, weight_grad = m.run_grad([loss_grad, feat, weight, labels, lse])

    ``loss_grad`` (n,) float32 is the gradient of whatever reduction of the losses the caller
    uses (1 / count for their mean).  A label out of range gives a loss of NaN, adds to no
    gradient and is reported by ``device_status``."""
    _compute_func = staticmethod(ops.softmax_cross_entropy)
    _schedule_func = staticmethod(ops.schedule_softmax_cross_entropy_cuda)

    def _allocate(self, out):
        feat, weight, labels = out.inputs
        self.out_tvm = self._own_zeros(out.shape, "float32")
        self.lse_tvm = self._own_zeros(out.shape, "float32")
        self.feat_grad_tvm = self.weight_grad_tvm = None
        if out.attrs["with_grad"]:
            self.feat_grad_tvm = self._own_zeros(feat.shape, feat.dtype)
            self.weight_grad_tvm = self._own_zeros(weight.shape, weight.dtype)
        self._codes = (_lib.DTYPES.index(feat.dtype), _lib.INDEX_TYPES.index(labels.dtype))

    def _workspace_bytes(self, out):
        return int(_lib.load().fg_softmax_xent_workspace_bytes(
            _lib.DTYPES.index(out.inputs[0].dtype), out.shape[0], out.attrs["vocab"],
            out.attrs["feat_len"], out.attrs["with_grad"]))

    def _checked_inputs(self, inputs):
        fp, wp, lp = self._spec.inputs
        return (self._tensor(inputs[0], fp.shape, fp.dtype, "Feat", rows=True),
                self._tensor(inputs[1], wp.shape, wp.dtype, "Weight", rows=True),
                self._tensor(inputs[2], lp.shape, lp.dtype, "Labels"))

    def _launch(self, feat, weight, labels):
        a = self._spec.attrs
        _lib.check(_lib.load().fg_softmax_xent(
            feat.data_ptr(), self._pitch(feat), weight.data_ptr(), self._pitch(weight),
            self._codes[0], labels.data_ptr(), self._codes[1], self._spec.shape[0], a["vocab"],
            a["feat_len"], a["scale"], a["ignore_index"], self.out_tvm.torch.data_ptr(),
            self.lse_tvm.torch.data_ptr(), self._workspace.data_ptr(), self._workspace_size,
            self._status.data_ptr(), self._ctx.device_id, self._stream()))

    def run(self, input_tvm_ndarrays):
        """[Feat, Weight, Labels] -> (``self.out_tvm``, ``self.lse_tvm``): the losses and the
        log-sum-exp of every row, the same arrays every call."""
        self._need(3, input_tvm_ndarrays, "run()")
        self._launch(*self._checked_inputs(input_tvm_ndarrays))
        return self.out_tvm, self.lse_tvm

    def measure_average_time(self, input_tvm_ndarrays, num_runs):
        """Mean seconds of the forward call over ``num_runs`` launches."""
        self._need(3, input_tvm_ndarrays, "measure_average_time()")
        inputs = self._checked_inputs(input_tvm_ndarrays)
        return time_launches(self._ctx, lambda: self._launch(*inputs), num_runs)

    def run_grad(self, input_tvm_ndarrays):
        """[LossGrad, Feat, Weight, Labels, Lse] -> (``self.feat_grad_tvm``,
        ``self.weight_grad_tvm``), the same arrays every call, every element overwritten.
        ``Lse`` is what ``run`` returned for these inputs."""
        self._need(5, input_tvm_ndarrays, "run_grad()")
        a = self._spec.attrs
        if not a["with_grad"]:
            raise RuntimeError("run_grad() needs build(..., {'with_grad': True}, ...)")
        dl = self._tensor(input_tvm_ndarrays[0], self._spec.shape, "float32", "LossGrad")
        feat, weight, labels = self._checked_inputs(input_tvm_ndarrays[1:4])
        lse = self._tensor(input_tvm_ndarrays[4], self._spec.shape, "float32", "Lse")
        _lib.check(_lib.load().fg_softmax_xent_grad(
            dl.data_ptr(), feat.data_ptr(), self._pitch(feat), weight.data_ptr(),
            self._pitch(weight), self._codes[0], labels.data_ptr(), self._codes[1],
            self._spec.shape[0], a["vocab"], a["feat_len"], a["scale"], a["ignore_index"],
            lse.data_ptr(), self.feat_grad_tvm.torch.data_ptr(),
            self.weight_grad_tvm.torch.data_ptr(), self._workspace.data_ptr(),
            self._workspace_size, self._status.data_ptr(), self._ctx.device_id, self._stream()))
        return self.feat_grad_tvm, self.weight_grad_tvm


class GradientClipcuda(_TrainingOp):
    """Global norm of many gradients and clipping.

        m = GradientClipcuda()
        m.build([Grad placeholders ...], {'max_norm': 1.0}, {})
        norm, clipped = m.run([grads ...])

    ``norm`` is a (1,) float32 array, ``clipped`` a list of arrays: the module's own, or with
    ``{'in_place': True}`` the inputs themselves.  ``{'norm_type': math.inf}`` takes the
    largest magnitude instead of the 2-norm."""
    _compute_func = staticmethod(ops.gradient_clip)
    _schedule_func = staticmethod(ops.schedule_gradient_clip_cuda)

    def _allocate(self, out):
        n = len(out.inputs)
        self.out_tvm = self._own_zeros((1,), "float32")
        self.clipped_tvm = None
        if not out.attrs["in_place"]:
            self.clipped_tvm = [self._own_zeros(p.shape, p.dtype) for p in out.inputs]
        sizes = [int(math.prod(p.shape)) for p in out.inputs]
        self._sizes = (ctypes.c_int64 * n)(*sizes)
        self._codes = (ctypes.c_int32 * n)(*[_lib.DTYPES.index(p.dtype) for p in out.inputs])
        self._ins = (ctypes.c_void_p * n)()
        if out.attrs["in_place"]:
            self._outs = self._ins
        else:
            self._outs = (ctypes.c_void_p * n)(*[a.torch.data_ptr() for a in self.clipped_tvm])

    def _workspace_bytes(self, out):
        return int(_lib.load().fg_gradient_clip_workspace_bytes(len(out.inputs)))

    def _launch(self, tensors):
        a = self._spec.attrs
        for k, t in enumerate(tensors):
            self._ins[k] = t.data_ptr()
        _lib.check(_lib.load().fg_gradient_clip(
            self._ins, self._outs, self._sizes, self._codes, len(tensors),
            a["norm_type"] == math.inf, a["max_norm"], a["eps"], self.out_tvm.torch.data_ptr(),
            self._workspace.data_ptr(), self._workspace_size, self._ctx.device_id,
            self._stream()))

    def _checked_inputs(self, inputs):
        self._need(len(self._spec.inputs) if self._spec else 0, inputs, "run()")
        tensors = [self._tensor(x, p.shape, p.dtype, "Grads[%d]" % k)
                   for k, (x, p) in enumerate(zip(inputs, self._spec.inputs))]
        if self._spec.attrs["in_place"]:
            spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size())
                           for t in tensors if t.numel())
            if any(b[0] < a[1] for a, b in zip(spans, spans[1:])):
                raise ValueError("two of the gradients share memory: in place they would be "
                                 "scaled twice")
        return tensors

    def run(self, input_tvm_ndarrays):
        """[Grads ...] -> (``self.out_tvm``, the clipped gradients)."""
        self._launch(self._checked_inputs(input_tvm_ndarrays))
        if self._spec.attrs["in_place"]:
            return self.out_tvm, list(input_tvm_ndarrays)
        return self.out_tvm, self.clipped_tvm

    def measure_average_time(self, input_tvm_ndarrays, num_runs):
        """Mean seconds per call over ``num_runs`` calls (in place, each clips again)."""
        tensors = self._checked_inputs(input_tvm_ndarrays)
        return time_launches(self._ctx, lambda: self._launch(tensors), num_runs)
