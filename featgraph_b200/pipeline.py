"""Calls put together: two host-buffer calls side by side (HostPair), and the training step of
a layer over a vertex embedding table (VertexPrediction).

Two independent host-buffer calls side by side:

``SpMMbase.run_host`` / ``SDDMMbase.run_host`` are synchronous: upload, launch, download,
wait.  Back to back, the host link idles while one call computes and the GPU idles while the
other one's result travels.  When the two calls do not depend on each other (the SpMM and the
SDDMM of one GNN layer read the same features) they can be issued from two host threads on
two CUDA streams, so that one call's transfers overlap the other's kernels and the link
carries uploads and downloads at the same time (PCIe is full duplex).  The C-ABI host
entry points release the interpreter lock while they wait, which is what lets two Python
threads do this.
"""
import threading
import time

import torch

from . import te
from .module import (EmbeddingLookupcuda, GradientClipcuda, SoftmaxCrossEntropycuda,
                     VanillaSpMMcuda)
from .runtime import NDArray


class HostPair(object):
    """Runs ``spmm.run_host(x_host, y_host)`` and ``sddmm.run_host(src_host, dst_host,
    out_host)`` concurrently, each on its own stream; ``run`` returns when both results are
    in host memory.  Single-GPU modules only (the sharded operators issue collectives, which
    must be enqueued in the same order on every rank)."""

    def __init__(self, spmm, sddmm):
        self.spmm, self.sddmm = spmm, sddmm
        self.device = spmm.ctx.torch_device
        self.streams = (torch.cuda.Stream(device=self.device),
                        torch.cuda.Stream(device=self.device))

    def _call(self, which, fn, args, errors, delay=0.0):
        try:
            if delay:
                time.sleep(delay)
            torch.cuda.set_device(self.device)
            with torch.cuda.stream(self.streams[which]):
                fn(*args)
        except BaseException as exc:        # handed to the caller's thread
            errors.append(exc)

    def run(self, x_host, y_host, src_host, dst_host, out_host):
        main = torch.cuda.current_stream(self.device)
        for s in self.streams:
            s.wait_stream(main)
        errors = []
        # The SDDMM call is the longer chain (two uploads, then a result of 4 bytes per edge to
        # bring back), so it is issued from this thread, at once: its uploads reach the copy
        # engine ahead of the SpMM's, whose thread holds its call back for a moment.
        t = threading.Thread(target=self._call,
                             args=(0, self.spmm.run_host, (x_host, y_host), errors, 3e-4))
        t.start()
        self._call(1, self.sddmm.run_host, (src_host, dst_host, out_host), errors)
        t.join()
        for s in self.streams:
            main.wait_stream(s)
        if errors:
            raise errors[0]
        return y_host, out_host


class VertexPrediction(object):
    """The gradient of one training step that predicts a vertex for every row of a sampled
    block, over one embedding table of all vertices (tied weights):

        x = scale * table[ids];  y = adj @ x;  loss_t = cross entropy of scale_out * y @ table^T
        at labels[t];  objective = mean of the losses of the rows that have a label

    ``adj`` (n_rows, n_cols) is the block's adjacency (scipy, float32), ``ids`` (n_cols,) names
    the vertex of each of its columns, ``labels`` (n_rows,) the vertex to predict, or
    ``ignore_index``.  ``run(table, ids, labels)`` returns (mean loss, norm, gradient): the
    table's gradient from both of its uses, clipped to ``max_norm``, and the norm it had
    before.  The arrays are the step's own, the same every call.  float32, as the SpMM is.
    The reference leaves the layers around its kernels to the caller (README.md:6)."""

    def __init__(self, adj_scipy, num_vertices, feat_len, scale=1.0, scale_out=1.0,
                 max_norm=float("inf"), ignore_index=-100, index_dtype="int64", device_id=0):
        adj = adj_scipy.tocsr()
        self.n_rows, self.n_cols = adj.shape
        self.ignore_index = int(ignore_index)
        self.forward = VanillaSpMMcuda(adj, device_id=device_id)
        self.backward = VanillaSpMMcuda(adj.T.tocsr(), device_id=device_id)
        self.lookup = EmbeddingLookupcuda(device_id)
        self.loss = SoftmaxCrossEntropycuda(device_id)
        self.clip = GradientClipcuda(device_id)
        table = te.placeholder((num_vertices, feat_len), "float32", "Table")
        self.forward.build([te.placeholder((self.n_cols, feat_len))], {}, {})
        self.backward.build([te.placeholder((self.n_rows, feat_len))], {}, {})
        self.lookup.build([table, te.placeholder((self.n_cols,), index_dtype)],
                          {"scale": scale, "with_grad": True}, {})
        self.loss.build([te.placeholder((self.n_rows, feat_len)), table,
                         te.placeholder((self.n_rows,), index_dtype)],
                        {"scale": scale_out, "ignore_index": ignore_index, "with_grad": True}, {})
        self.clip.build([table], {"max_norm": max_norm, "in_place": True}, {})

    def run(self, table, ids, labels):
        x = self.lookup.run([table, ids])
        y = self.forward.run([x])
        losses, lse = self.loss.run([y, table, labels])
        wanted = labels.torch if isinstance(labels, NDArray) else labels
        live = (wanted != self.ignore_index).to(torch.float32)
        share = live / live.sum().clamp(min=1.0)
        y_grad, grad = self.loss.run_grad([share, y, table, labels, lse])
        x_grad = self.backward.run([y_grad])
        self.lookup.run_grad([x_grad, ids], accumulate_into=grad)
        norm, (grad,) = self.clip.run([grad])
        return (losses.torch * share).sum(), norm, grad

    def device_status(self):
        """Synchronise; raises if an id or a label was out of range or a wait gave up."""
        for m in (self.forward, self.backward, self.lookup, self.loss):
            m.device_status()
        return 0
