"""Op layer of the training operators: the vertex embedding lookup, the softmax cross entropy
over a large vocabulary and the gradient clip.  The reference has no counterpart (it stops at
SpMM and SDDMM, python/featgraph/op/__init__.py:1-5); names, placeholders and the split into a
compute and a schedule function follow its ops."""
import math

from .spec import ComputeSpec, ScheduleSpec
from .._lib import DTYPES, INDEX_TYPES


def _check_dtype(p, what):
    if p.dtype not in DTYPES:
        raise TypeError("%s: dtype must be one of %r, got %s" % (what, DTYPES, p.dtype))


def _check_index(p, what):
    if p.dtype not in INDEX_TYPES:
        raise TypeError("%s: dtype must be one of %r, got %s" % (what, INDEX_TYPES, p.dtype))
    if len(p.shape) != 1:
        raise ValueError("%s must be 1-D, got %r" % (what, p.shape))


def _check_matrix(p, what):
    _check_dtype(p, what)
    if len(p.shape) != 2 or p.shape[1] < 1:
        raise ValueError("%s must be 2-D with at least one column, got %r" % (what, p.shape))


def _finite(x, what):
    x = float(x)
    if not math.isfinite(x):
        raise ValueError("%s must be finite, got %r" % (what, x))
    return x


def _finite32(x, what):
    """A number that reaches the kernels as float32."""
    x = _finite(x, what)
    if abs(x) >= 2.0 ** 128 - 2.0 ** 103:      # rounds to infinity there
        raise ValueError("%s must be finite as float32, got %r" % (what, x))
    return x


def embedding_lookup(Table, Ids, scale=1.0, padding_idx=None, with_grad=False):
    """Out[i, f] = scale * Table[Ids[i], f], rounded once to the table's type.

    Table : placeholder, (num_vertices, feat_len), float32 / bfloat16 / float16
    Ids : placeholder, (num_ids,), int32 / int64; any order, any repeats
    scale : a number
    padding_idx : the vertex that receives no gradient (its row is looked up like any other)
    with_grad : whether the module's ``run_grad`` will be used (it owns the table's gradient)
    """
    _check_matrix(Table, "Table")
    _check_index(Ids, "Ids")
    if padding_idx is not None:
        padding_idx = int(padding_idx)
        if not 0 <= padding_idx < Table.shape[0]:
            raise ValueError("padding_idx %d is not a row of a table of %d rows"
                             % (padding_idx, Table.shape[0]))
    return ComputeSpec("embedding_lookup", (Ids.shape[0], Table.shape[1]), Table.dtype,
                       (Table, Ids),
                       {"scale": _finite32(scale, "scale"), "padding_idx": padding_idx,
                        "with_grad": bool(with_grad), "num_vertices": Table.shape[0],
                        "feat_len": Table.shape[1]})


def schedule_embedding_lookup_cuda(Out):
    """The launch shapes follow from the sizes; there are no knobs."""
    return ScheduleSpec(Out, "cuda", {})


def softmax_cross_entropy(Feat, Weight, Labels, scale=1.0, ignore_index=-100, with_grad=False):
    """Loss[t] = log sum_v exp Z[t, v] - Z[t, Labels[t]] with Z = scale * Feat @ Weight^T,
    which is never stored; 0 where Labels[t] is ``ignore_index``.

    Feat : placeholder, (num_samples, feat_len), float32 / bfloat16 / float16
    Weight : placeholder, (num_vertices or num_classes, feat_len), the same type
    Labels : placeholder, (num_samples,), int32 / int64
    with_grad : whether the module's ``run_grad`` will be used (it owns both gradients)
    """
    _check_matrix(Feat, "Feat")
    _check_matrix(Weight, "Weight")
    _check_index(Labels, "Labels")
    if Feat.dtype != Weight.dtype:
        raise TypeError("Feat is %s, Weight is %s" % (Feat.dtype, Weight.dtype))
    assert Feat.shape[1] == Weight.shape[1], "dimension mismatch"
    assert Feat.shape[0] == Labels.shape[0], "dimension mismatch"
    if Weight.shape[0] < 1:
        raise ValueError("Weight needs at least one row")
    ignore_index = int(ignore_index)
    if not -2 ** 63 <= ignore_index < 2 ** 63:
        raise ValueError("ignore_index %d does not fit 64 bits" % ignore_index)
    return ComputeSpec("softmax_cross_entropy", (Feat.shape[0],), "float32",
                       (Feat, Weight, Labels),
                       {"scale": _finite32(scale, "scale"), "ignore_index": ignore_index,
                        "with_grad": bool(with_grad), "vocab": Weight.shape[0],
                        "feat_len": Feat.shape[1]})


def schedule_softmax_cross_entropy_cuda(Out):
    """The tiles and pieces follow from the sizes; there are no knobs."""
    return ScheduleSpec(Out, "cuda", {})


def gradient_clip(*Grads, max_norm=math.inf, norm_type=2, eps=1e-6, in_place=False):
    """Norm = (sum over all elements of all Grads of g^2)^(1/2), or max |g| with
    ``norm_type=math.inf``; Clipped_k = Grads_k * min(1, max_norm / (Norm + eps)).

    Grads : placeholders of any shapes, float32 / bfloat16 / float16, also mixed
    max_norm : the bound; infinite (the default) computes the norm and scales by 1
    in_place : write the results over the inputs instead of into the module's own arrays
    """
    for k, g in enumerate(Grads):
        _check_dtype(g, "Grads[%d]" % k)
    max_norm, eps = float(max_norm), _finite(eps, "eps")
    if not max_norm >= 0 or eps < 0:
        raise ValueError("max_norm and eps must not be negative, got %r and %r" % (max_norm, eps))
    if norm_type not in (2, 2.0, math.inf):
        raise ValueError("norm_type must be 2 or math.inf, got %r" % (norm_type,))
    return ComputeSpec("gradient_clip", (1,), "float32", Grads,
                       {"max_norm": max_norm, "norm_type": float(norm_type), "eps": eps,
                        "in_place": bool(in_place)})


def schedule_gradient_clip_cuda(Out):
    """The launch shapes follow from the sizes; there are no knobs."""
    return ScheduleSpec(Out, "cuda", {})
