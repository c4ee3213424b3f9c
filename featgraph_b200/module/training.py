"""Module classes of the training operators, with the interface of the SpMM and SDDMM modules
(``build`` fixes the shapes and allocates the outputs, ``run`` launches and returns the same
arrays every call): the vertex embedding lookup that feeds an SpMM, the softmax cross entropy
that reads its output, and the gradient clip before the optimiser.  The reference has no
counterpart (python/featgraph/module/__init__.py:1-2).

A module's outputs and workspace are shared state: one call at a time per module.  Its outputs
are not its inputs: an array that shares memory with one is refused (a gradient clip takes the
array that it writes to as its own input).  A call on
another stream than the module's last one waits for that one first.  While a stream is being
captured nothing is waited for, and of a graph's replays a module knows nothing: two graphs that
hold calls of one module must not be replayed side by side, nor a replay beside a call of the
module on another stream, and a module that a graph holds calls of stays alive until the graph is
gone (its outputs and workspace are the module's memory; building the module again keeps them).
"""
import array
import math
import struct

import torch

from .. import _lib
from ..op import training as ops
from ..runtime import NDArray, gpu, zeros
from .base import time_launches

_TORCH_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16,
                 "int32": torch.int32, "int64": torch.int64}


# The argument words of the C calls (fg_training_call): q an integer or a pointer, d a number.
_LOOKUP = struct.Struct("=8qd5q")
_LOOKUP_GRAD = struct.Struct("=8qd8q")
_XENT = struct.Struct("=10qd8q")
_XENT_GRAD = struct.Struct("=11qd9q")
_CLIP = struct.Struct("=6qdd5q")


class _TrainingOp(object):
    """What the three modules share: device, workspace, status word, stream hand-over."""
    _compute_func = None
    _schedule_func = None

    def __init__(self, device_id=0):
        if not torch.cuda.is_available():
            raise RuntimeError("%s needs a CUDA device; there is no CPU fallback"
                               % type(self).__name__)
        self._target = "cuda"
        self._call = _lib.load().fg_training_call
        self._ctx = gpu(int(device_id))
        self._device = self._ctx.torch_device
        self._index = self._ctx.device_id
        self._spec = None
        self._owned, self._captured, self._of_graphs = [], False, []
        self.out_tvm = None

    def _specialise(self, input_placeholders, compute_args, schedule_args):
        out = type(self)._compute_func(*input_placeholders, **compute_args)
        return out, type(self)._schedule_func(out, **schedule_args)

    def build(self, input_placeholders, compute_args, schedule_args):
        """Fix the static shapes; allocate the outputs and the workspace."""
        out, _ = self._specialise(input_placeholders, compute_args, schedule_args)
        self._spec = None
        if self._captured:
            self._of_graphs.append(self._owned)     # replays still write there
        self._owned, self._captured = [], False
        self._status = self._own(torch.zeros(1, dtype=torch.int32, device=self._device))
        self._allocate(out)
        self._take_workspace(self._workspace_bytes(out))
        self._status_at = self._status.data_ptr()
        self._last_stream = torch.cuda.current_stream(self._device)
        self._last_handle = self._last_stream.cuda_stream
        self._spec = out

    def _take_workspace(self, size):
        size = max(size, 16)
        workspace = self._own(torch.empty(size, dtype=torch.uint8, device=self._device))
        self._workspace_size, self._workspace_at = size, workspace.data_ptr()

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
        handle = torch._C._cuda_getCurrentRawStream(self._index)
        if handle:                                  # 0: the default stream, which nothing captures
            self._captured = self._captured or self._is_capturing()
        if handle != self._last_handle:
            self._change_stream(handle)
        return handle

    def _is_capturing(self):
        if torch._C._cuda_getDevice() == self._index:
            return torch._C._cuda_isCurrentStreamCapturing()
        with torch.cuda.device(self._device):       # whose current stream the handle is
            return torch.cuda.is_current_stream_capturing()

    def _change_stream(self, handle):
        if handle and self._is_capturing():
            return
        stream = torch.cuda.current_stream(self._device)
        stream.wait_stream(self._last_stream)
        for t in self._owned:
            t.record_stream(stream)
        self._last_stream, self._last_handle = stream, handle

    def _need(self, count, inputs, what):
        if self._spec is None:
            raise RuntimeError("build() must be called before %s" % what)
        if len(inputs) != count:
            raise ValueError("%s takes exactly %d input arrays, got %d" % (what, count, len(inputs)))

    @staticmethod
    def _expect(placeholder, what, rows=False, dtype=None):
        """What ``_tensor`` checks an input against; ``rows``: a 2-D array whose rows may lie
        apart (each row itself contiguous)."""
        return (placeholder.shape, _TORCH_DTYPES[dtype or placeholder.dtype], what, rows)

    def _tensor(self, x, expected):
        """One input as a torch tensor, checked (this runs in every call: the usual case is
        one line)."""
        t = x.torch if type(x) is NDArray else x
        if isinstance(t, torch.Tensor) and t.dtype is expected[1] and t.shape == expected[0] \
                and t.get_device() == self._index and t.is_contiguous():
            return t
        return self._odd_tensor(x, *expected)

    def _odd_tensor(self, x, shape, dtype, what, rows):
        t = x.torch if isinstance(x, NDArray) else x
        if not isinstance(t, torch.Tensor):
            raise TypeError("%s: expected an NDArray or a torch.Tensor, got %r" % (what, type(x)))
        if t.dtype != dtype:
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
    def _meet(a, b):
        """Whether two tensors have memory in common (rows that lie apart count with their gaps)."""
        def span(t):
            last = sum((n - 1) * s for n, s in zip(t.shape, t.stride())) if t.numel() else -1
            return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()
        (a0, a1), (b0, b1) = span(a), span(b)
        return a0 < b1 and b0 < a1

    def _rows(self, x, expected):
        """``_tensor`` and the distance between its rows in elements."""
        t = self._tensor(x, expected)
        width = expected[0][1]
        return t, width if t.is_contiguous() or expected[0][0] < 2 else t.stride(0)

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
        self._table = self._expect(table, "Table", rows=True)
        self._ids = self._expect(ids, "Ids")
        self._into = self._expect(table, "accumulate_into")
        self._out_grad = (out.shape, self._table[1], "OutGrad", True)
        a = out.attrs
        self._sizes = (out.shape[0], a["num_vertices"], a["feat_len"], a["scale"])
        self._padding = -1 if a["padding_idx"] is None else a["padding_idx"]
        self._out_at = self.out_tvm.torch.data_ptr()

    def _workspace_bytes(self, out):
        if not out.attrs["with_grad"]:
            return 0
        return int(_lib.load().fg_embedding_grad_workspace_bytes(
            out.shape[0], out.attrs["num_vertices"], out.attrs["feat_len"]))

    def _launch(self, table, pitch, ids):
        n, vertices, feat_len, scale = self._sizes
        code = self._call(_lib.OP_LOOKUP, _LOOKUP.pack(
            table.data_ptr(), self._codes[0], pitch, vertices, ids.data_ptr(), self._codes[1], n,
            feat_len, scale, self._out_at, feat_len, self._status_at, self._index,
            self._stream()), 14)
        if code:
            _lib.check(code)

    def _checked_inputs(self, inputs):
        self._need(2, inputs, "run()")
        return self._rows(inputs[0], self._table) + (self._tensor(inputs[1], self._ids),)

    def run(self, input_tvm_ndarrays):
        """[Table, Ids] -> ``self.out_tvm``, the same array every call."""
        self._launch(*self._checked_inputs(input_tvm_ndarrays))
        return self.out_tvm

    def measure_average_time(self, input_tvm_ndarrays, num_runs):
        """Mean seconds of the lookup over ``num_runs`` launches."""
        inputs = self._checked_inputs(input_tvm_ndarrays)
        return time_launches(self._ctx, lambda: self._launch(*inputs), num_runs)

    def run_grad(self, input_tvm_ndarrays, accumulate_into=None):
        """[OutGrad (n, F), Ids] -> the table's gradient (V, F): ``self.grad_tvm``, the same
        array every call, every element overwritten.  ``accumulate_into``: a contiguous (V, F)
        array of the table's type (say, the gradient that a loss with tied weights left) that
        the sums are added onto instead; it is returned."""
        self._need(2, input_tvm_ndarrays, "run_grad()")
        if self.grad_tvm is None:
            raise RuntimeError("run_grad() needs build(..., {'with_grad': True}, ...)")
        dy, pitch = self._rows(input_tvm_ndarrays[0], self._out_grad)
        ids = self._tensor(input_tvm_ndarrays[1], self._ids)
        if accumulate_into is None:
            result, grad = self.grad_tvm, self.grad_tvm.torch
        else:
            result, grad = accumulate_into, self._tensor(accumulate_into, self._into)
            if self._meet(grad, dy):
                raise ValueError("OutGrad and accumulate_into share memory")
        n, vertices, feat_len, scale = self._sizes
        code = self._call(_lib.OP_LOOKUP_GRAD, _LOOKUP_GRAD.pack(
            dy.data_ptr(), self._codes[0], pitch, ids.data_ptr(), self._codes[1], n, vertices,
            feat_len, scale, self._padding, accumulate_into is not None, grad.data_ptr(),
            self._workspace_at, self._workspace_size, self._status_at, self._index,
            self._stream()), 17)
        if code:
            _lib.check(code)
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
        self._inputs = (self._expect(feat, "Feat", rows=True),
                        self._expect(weight, "Weight", rows=True), self._expect(labels, "Labels"))
        self._loss_grad = (out.shape, torch.float32, "LossGrad", False)
        self._lse = (out.shape, torch.float32, "Lse", False)
        a = out.attrs
        self._sizes = (out.shape[0], a["vocab"], a["feat_len"], a["scale"], a["ignore_index"])
        self._has_room = feat.dtype == "float32" or a["feat_len"] % 8 != 0   # for a packed table
        self._loss_at, self._lse_at = self.out_tvm.torch.data_ptr(), self.lse_tvm.torch.data_ptr()

    def _workspace_bytes(self, out, in_place=None):
        """``in_place``: for a table that needs no packed copy; by default, whether a contiguous
        table of these sizes is one."""
        if in_place is None:
            in_place = out.inputs[1].dtype != "float32" and out.attrs["feat_len"] % 8 == 0
        return int(_lib.load().fg_softmax_xent_workspace_bytes(
            _lib.DTYPES.index(out.inputs[0].dtype), out.shape[0], out.attrs["vocab"],
            out.attrs["feat_len"], out.attrs["with_grad"] + (_lib.XENT_TABLE_IN_PLACE if in_place else 0)))

    def _checked_inputs(self, inputs):
        e = self._inputs
        weight, pitch = self._rows(inputs[1], e[1])
        if (pitch & 7 or weight.data_ptr() & 15) and not self._has_room:
            self._stream()                     # ordered behind the calls that use the smaller one
            self._take_workspace(self._workspace_bytes(self._spec, in_place=False))
            self._has_room = True
        return self._rows(inputs[0], e[0]) + (weight, pitch, self._tensor(inputs[2], e[2]))

    def _launch(self, feat, feat_pitch, weight, weight_pitch, labels):
        n, vocab, feat_len, scale, ignore = self._sizes
        code = self._call(_lib.OP_XENT, _XENT.pack(
            feat.data_ptr(), feat_pitch, weight.data_ptr(), weight_pitch, self._codes[0],
            labels.data_ptr(), self._codes[1], n, vocab, feat_len, scale, ignore, self._loss_at,
            self._lse_at, self._workspace_at, self._workspace_size, self._status_at, self._index,
            self._stream()), 19)
        if code:
            _lib.check(code)

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
        if self.feat_grad_tvm is None:
            raise RuntimeError("run_grad() needs build(..., {'with_grad': True}, ...)")
        dl = self._tensor(input_tvm_ndarrays[0], self._loss_grad)
        feat, feat_pitch, weight, weight_pitch, labels = \
            self._checked_inputs(input_tvm_ndarrays[1:4])
        lse = self._tensor(input_tvm_ndarrays[4], self._lse)
        n, vocab, feat_len, scale, ignore = self._sizes
        code = self._call(_lib.OP_XENT_GRAD, _XENT_GRAD.pack(
            dl.data_ptr(), feat.data_ptr(), feat_pitch, weight.data_ptr(), weight_pitch,
            self._codes[0], labels.data_ptr(), self._codes[1], n, vocab, feat_len, scale, ignore,
            lse.data_ptr(), self.feat_grad_tvm.torch.data_ptr(),
            self.weight_grad_tvm.torch.data_ptr(), self._workspace_at, self._workspace_size,
            self._status_at, self._index, self._stream()), 21)
        if code:
            _lib.check(code)
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
        # host arrays of the C call; what address they lie at is asked for once
        self._sizes = array.array("q", [int(math.prod(p.shape)) for p in out.inputs] or [0])
        self._codes = array.array("i", [_lib.DTYPES.index(p.dtype) for p in out.inputs] or [0])
        self._outs = None
        if not out.attrs["in_place"]:
            self._outs = array.array("Q", [a.torch.data_ptr() for a in self.clipped_tvm] or [0])
            self._outs_at = self._outs.buffer_info()[0]
        self._sizes_at, self._codes_at = (a.buffer_info()[0] for a in (self._sizes, self._codes))
        self._inputs = [self._expect(p, "Grads[%d]" % k) for k, p in enumerate(out.inputs)]
        self._args = (n, out.attrs["norm_type"] == math.inf, out.attrs["max_norm"],
                      out.attrs["eps"], self.out_tvm.torch.data_ptr())

    def _workspace_bytes(self, out):
        return int(_lib.load().fg_gradient_clip_workspace_bytes(len(out.inputs)))

    def _launch(self, tensors):
        ins = array.array("Q", [t.data_ptr() for t in tensors])
        ins_at = ins.buffer_info()[0]
        code = self._call(_lib.OP_CLIP, _CLIP.pack(
            ins_at, ins_at if self._outs is None else self._outs_at, self._sizes_at,
            self._codes_at, *self._args, self._workspace_at, self._workspace_size, self._index,
            self._stream()), 13)
        if code:
            _lib.check(code)

    def _checked_inputs(self, inputs):
        self._need(len(self._spec.inputs) if self._spec else 0, inputs, "run()")
        tensors = [self._tensor(x, e) for x, e in zip(inputs, self._inputs)]
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
