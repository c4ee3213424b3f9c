"""Edges of the training operators on the GPU: operands whose rows lie far apart in size, masked
and infinite rows, ignored rows.  Plain implementations in 64 bits, as in
test_training_ops_gpu.py."""
import math

import pytest
import torch

from featgraph_b200 import _lib, module, nd, te
import test_training_ops_gpu as t

pytestmark = pytest.mark.gpu
U = t.U


# ------------------------------------- float32 cross entropy: rows of any size --
def by_rows(feat, weight, labels, dloss, scale=1.0, ignore=-100):
    """Losses and gradients in fp64 with the bounds of float32 held as two fp16 pieces relative to
    the largest value of its OWN row.

    An element x of a row whose largest magnitude is m is off by at most 2^-22 |x| + 2^-37 m (the
    second piece is rounded to 2^-11 of the first's error, and ends at 2^-24 where m is at least
    2^12); a product leaves out the two second pieces, 2^-22.  Sums as in xent_reference: 2 u a
    term.  dz is held in two pieces relative to the largest entry of its row so far (probability
    times the scale of the row that it multiplies), which is held as at least 2^13.  Each piece ends
    at 2^-24, half a step of it is 2^-25, and where a larger entry comes both are rounded again at
    half the size or less: 2^-23 in all.  The rows that they multiply are below 2^13, and the
    largest contribution at least 2^13 2^12: k terms are off by k 2^-35 of that.  Nothing is
    relative to the values of another row beside the largest contribution."""
    h, w = feat.double(), weight.double()
    n, d = h.shape
    v = w.shape[0]
    keep = labels != ignore
    hm, wm = h.abs().amax(1, keepdim=True), w.abs().amax(1, keepdim=True)
    z = scale * (h @ w.T)
    ends = (h.abs().sum(1, keepdim=True) @ wm.T + hm @ w.abs().sum(1, keepdim=True).T) * 2.0 ** -37
    ez = abs(scale) * ((h.abs() @ w.abs().T) * ((d + 8) * 2 * U + 2.0 ** -20) + ends)
    lse = torch.logsumexp(z, 1)
    p = torch.exp(z - lse[:, None])
    # a logit's error counts by its probability, within the largest of those that count at all
    far = z + ez < (z - ez).amax(1, keepdim=True) - 120
    elz = torch.where(far, 0.0, ez).amax(1) + (v + 64) * U + lse.abs() * 4 * U
    at = torch.where(keep, labels.long(), 0)[:, None]
    loss = torch.where(keep, lse - z.gather(1, at)[:, 0], 0.0)
    eloss = torch.where(keep, elz + ez.gather(1, at)[:, 0] + loss.abs() * 2 * U, 0.0)
    g = torch.where(keep, dloss.double(), 0.0)[:, None]
    hot = torch.zeros_like(p).scatter_(1, at, 1.0)
    dz = (p - hot) * g * scale
    ep = torch.where(far, 0.0, p * (torch.expm1(ez.clamp(max=300) + elz.clamp(max=300)[:, None]) + 16 * U))
    ep = ep * (g * scale).abs()
    edz = ep + (dz.abs() + ep) * 2.0 ** -20
    unit = torch.maximum(p, hot) * (g * scale).abs()
    hk = torch.where(keep[:, None], h, 0.0)
    hmk = torch.where(keep[:, None], hm, 0.0)
    size = dz.abs()
    df = edz @ w.abs() + (size @ w.abs()) * ((v + 8) * 2 * U + 2.0 ** -20) + (size @ wm) * 2.0 ** -37
    df = df + (unit * wm.T).amax(1, keepdim=True) * v * 2.0 ** -35
    dw = edz.T @ hk.abs() + (size.T @ hk.abs()) * ((n + 8) * 2 * U + 2.0 ** -20) + (size.T @ hmk) * 2.0 ** -37
    dw = dw + (unit * hmk).amax(0)[:, None] * n * 2.0 ** -35
    return {"loss": (loss, eloss), "lse": (lse, elz),
            "feat_grad": (torch.where(keep[:, None], dz @ w, 0.0), torch.where(keep[:, None], df, 0.0)),
            "weight_grad": (dz.T @ hk, dw)}


def run(m, feat, weight, labels, dloss):
    loss, lse = m.run([feat, weight, labels])
    dh, dw = m.run_grad([dloss, feat, weight, labels, lse])
    return {"loss": loss.torch, "lse": lse.torch, "feat_grad": dh.torch, "weight_grad": dw.torch}


def check_rows(feat, weight, labels, dloss, scale=1.0, rows=slice(None), vertices=slice(None)):
    got = run(t.xent_module(feat, weight, labels, scale=scale), feat, weight, labels, dloss)
    want = by_rows(feat, weight, labels, dloss, scale)
    pick = {"loss": rows, "lse": rows, "feat_grad": rows, "weight_grad": vertices}
    for key, (value, bound) in want.items():
        t.check(got[key][pick[key]], value[pick[key]], bound[pick[key]], torch.float32)
    return got


SIZES = [(60, 400, 40), (150, 700, 128), (33, 300, 260)]      # one tile a row, two, streamed


@pytest.mark.parametrize("n, v, d", SIZES)
@pytest.mark.parametrize("mask", [-1e6, -1e9, torch.finfo(torch.float32).min])
def test_float32_masked_table_rows_leave_the_others_alone(n, v, d, mask):
    # a column of ones in the features carries the mask
    feat, weight, labels, dloss = t.xent_inputs(n, v, d, "float32", n + d)
    feat[:, 0] = 1.0
    for row in (5, 133, v - 1):
        weight[row] = 0.0
        weight[row, 0] = mask
        labels[labels == row] = 6
    check_rows(feat, weight, labels, dloss)


@pytest.mark.parametrize("n, v, d", SIZES)
@pytest.mark.parametrize("size", [2.0 ** 24, 1e7, 1e-7])
def test_float32_one_sample_of_another_size(n, v, d, size):
    feat, weight, labels, dloss = t.xent_inputs(n, v, d, "float32", n + d + 1)
    labels[7] = 3
    feat[7] *= size
    best = int((feat[7].double() @ weight.double().T).argmax())
    rest = [i for i in range(n) if i != 7]
    check_rows(feat, weight, labels, dloss, rows=rest,
               vertices=[i for i in range(v) if i not in (3, best)])


@pytest.mark.parametrize("n, v, d", SIZES)
def test_float32_one_table_row_of_another_size(n, v, d):
    # a large row that no sample comes near: its features point away from it
    feat, weight, labels, dloss = t.xent_inputs(n, v, d, "float32", n + d + 2)
    feat[:, 0] = 1.0 + feat[:, 0].abs()
    weight[9, 0] = -2.0 ** 24
    labels[labels == 9] = 10
    weight[11] *= 2.0 ** -30
    labels[0] = 11
    check_rows(feat, weight, labels, dloss)


@pytest.mark.parametrize("n, v, d", SIZES)
@pytest.mark.parametrize("size", [100.0, 1e3, 1e6, 1e-6])
def test_float32_lse_of_ignored_rows_is_theirs(n, v, d, size):
    feat, weight, labels, dloss = t.xent_inputs(n, v, d, "float32", n + d + 3)
    labels[4] = labels[20] = -100
    feat[4] *= size
    check_rows(feat, weight, labels, dloss)


@pytest.mark.parametrize("size", [1e-6, 1e-5, 1e5, 1e6])
def test_float32_lse_where_every_row_is_ignored(size):
    feat, weight, labels, dloss = t.xent_inputs(70, 333, 48, "float32", 4)
    labels.fill_(-100)
    got = check_rows(feat * size, weight / size, labels, dloss)
    assert not got["loss"].any() and not got["feat_grad"].any() and not got["weight_grad"].any()


@pytest.mark.parametrize("n, v, d", SIZES)
@pytest.mark.parametrize("scale", [1.0, -0.5])
def test_float32_minus_infinity_in_table_rows(n, v, d, scale):
    # such a vertex has probability 0: losses, the table's gradient and (but for the columns that
    # hold an infinity, where 0 times it is NaN) the features' are those of the other vertices
    feat, weight, labels, dloss = t.xent_inputs(n, v, d, "float32", n + d + 5)
    feat[:, 0] = feat[:, 2] = math.copysign(1.0, scale)
    gone = [5, 130, v - 1]
    for row in gone:
        labels[labels == row] = 6
    kept = [i for i in range(v) if i not in gone]
    place = torch.zeros(v, dtype=torch.int64, device="cuda")
    place[kept] = torch.arange(len(kept), device="cuda")
    small = torch.where(labels == -100, labels, place[labels.clamp(min=0)])
    want = by_rows(feat, weight[kept], small, dloss, scale)
    weight[5, 0] = weight[130, 2] = -math.inf
    weight[v - 1, 0] = weight[v - 1, 2] = -math.inf
    got = run(t.xent_module(feat, weight, labels, scale=scale), feat, weight, labels, dloss)
    for key in ("loss", "lse"):
        t.check(got[key], *want[key], torch.float32)
    t.check(got["weight_grad"][kept], *want["weight_grad"], torch.float32)
    assert not got["weight_grad"][gone].any()
    cols = [c for c in range(d) if c not in (0, 2)]
    t.check(got["feat_grad"][:, cols], want["feat_grad"][0][:, cols], want["feat_grad"][1][:, cols],
            torch.float32)
    dead = labels == -100
    assert got["feat_grad"][~dead][:, [0, 2]].isnan().all() and not got["feat_grad"][dead].any()


@pytest.mark.parametrize("n, v, d", [(200, 900, 128), (70, 600, 260), (9, 300, 1)])
@pytest.mark.parametrize("share", [0.1, 0.9])
def test_float32_many_masked_vertices(n, v, d, share):
    # candidates left out by one column, the last or another, or by a whole row
    feat, weight, labels, dloss = t.xent_inputs(n, v, d, "float32", n + d + 7)
    feat = feat.abs() + 0.1
    g = t.gen(5)
    gone = torch.rand(v, generator=g, device="cuda") < share
    gone[0] = False
    at = torch.randint(d, (v,), generator=g, device="cuda")
    at[::3] = d - 1
    whole = torch.rand(v, generator=g, device="cuda") < 0.2
    labels = torch.where((labels >= 0) & gone[labels.clamp(min=0)], 0, labels)
    kept = (~gone).nonzero()[:, 0]
    place = torch.zeros(v, dtype=torch.int64, device="cuda")
    place[kept] = torch.arange(len(kept), device="cuda")
    want = by_rows(feat, weight[kept], torch.where(labels == -100, labels, place[labels.clamp(min=0)]), dloss)
    weight[gone, at[gone]] = -math.inf
    weight[gone & whole] = -math.inf
    got = run(t.xent_module(feat, weight, labels), feat, weight, labels, dloss)
    for key in ("loss", "lse"):
        t.check(got[key], *want[key], torch.float32)
    t.check(got["weight_grad"][kept], *want["weight_grad"], torch.float32)
    assert not got["weight_grad"][gone].any()


def test_float32_infinities_and_nan_stay_in_their_samples():
    # a sample with an infinity or a NaN is NaN itself; a NaN in the table is everybody's
    feat, weight, labels, dloss = t.xent_inputs(140, 300, 72, "float32", 21)
    labels[3] = labels[4] = 8
    clean = {k: x.clone() for k, x in run(t.xent_module(feat, weight, labels), feat, weight, labels,
                                          dloss).items()}
    feat[3, 5], feat[4, 70] = math.inf, math.nan
    got = run(t.xent_module(feat, weight, labels), feat, weight, labels, dloss)
    rest = [i for i in range(140) if i not in (3, 4)]
    for key in ("loss", "lse", "feat_grad"):
        assert got[key][[3, 4]].isnan().all() and torch.equal(got[key][rest], clean[key][rest])
    assert got["weight_grad"].isnan().all()
    labels[3] = labels[4] = -100
    got = run(t.xent_module(feat, weight, labels), feat, weight, labels, dloss)
    assert got["lse"][[3, 4]].isnan().all() and not got["weight_grad"].isnan().any()
    weight[290, 1] = math.nan
    got = run(t.xent_module(feat, weight, labels), feat, weight, labels, dloss)
    assert got["lse"].isnan().all()


@pytest.mark.parametrize("n, v, d", SIZES)
@pytest.mark.parametrize("size", [1.0, 2.0 ** -40])
def test_float32_rows_of_zeros_take_nothing_from_the_others(n, v, d, size):
    # vertices that nothing has trained yet, samples without neighbours: their probabilities are as
    # large as any, and what they multiply is zero
    feat, weight, labels, dloss = t.xent_inputs(n, v, d, "float32", n + d + 6)
    weight[::3] = 0.0
    weight[v - 1] = 0.0
    feat[::4] = 0.0
    labels[1], labels[4] = 3, v - 1                       # also as labels
    check_rows(feat, weight * size, labels, dloss, scale=1.0 / size)
    check_rows(feat * size, weight, labels, dloss, scale=1.0 / size)


def test_float32_loss_gradients_of_any_size():
    # each sample's weight is its own: a large one takes nothing from the others' gradients
    feat, weight, labels, dloss = t.xent_inputs(200, 500, 64, "float32", 22)
    labels[9] = 17
    dloss[9] = 1e9
    feat[9] = 0.0
    feat[9, 0] = 1.0
    for row in (30, 31):
        dloss[row] = 1e-12
    want = by_rows(feat, weight, labels, dloss)
    got = run(t.xent_module(feat, weight, labels), feat, weight, labels, dloss)
    t.check(got["feat_grad"], *want["feat_grad"], torch.float32)
    # the large sample has one feature only: the table's other columns are the others' alone
    value, bound = want["weight_grad"]
    t.check(got["weight_grad"], value, bound, torch.float32)


# ------------------------------------------------------------ losses below zero --
@pytest.mark.parametrize("dtype", sorted(t.TYPES))
@pytest.mark.parametrize("n, v, d, size", [(3000, 40, 64, 3.0), (600, 2000, 100, 2.0)])
def test_no_loss_is_below_zero(dtype, n, v, d, size):
    # samples that point at their own label's row: lse and the label's logit agree to the last bits
    g = t.gen(n)
    weight = torch.randn((v, d), generator=g, device="cuda").to(t.TYPES[dtype])
    labels = torch.randint(v, (n,), generator=g, device="cuda")
    feat = (weight[labels].float() * size).to(weight.dtype)
    m = t.xent_module(feat, weight, labels)
    loss = m.run([feat, weight, labels])[0].torch
    assert not loss.isnan().any() and (loss >= 0).all() and (loss == 0).any()
    labels[5] = v
    loss = m.run([feat, weight, labels])[0].torch
    assert loss[5].isnan() and int(loss.isnan().sum()) == 1
    with pytest.raises(_lib.FeatGraphError, match="out of range"):
        m.device_status()


# ------------------------------------------------------------------ the status word --
def test_an_expired_wait_is_not_hidden_by_an_index_out_of_range():
    # the word as a kernel leaves it that gave up a wait; every later call meets a bad index
    table = torch.randn((10, 8), device="cuda")
    bad = torch.tensor([3, 10, -1], device="cuda")
    many = torch.full((9000,), 10, device="cuda")
    e, big, c = (module.EmbeddingLookupcuda(), module.EmbeddingLookupcuda(),
                 module.SoftmaxCrossEntropycuda())
    e.build(t.like(table, bad), {"with_grad": True}, {})
    big.build(t.like(table, many), {"with_grad": True}, {})
    c.build(t.like(table[:3], table, bad), {"with_grad": True}, {})
    loss = torch.zeros(3, device="cuda")
    calls = [(e, lambda: e.run([table, bad])),
             (e, lambda: e.run_grad([table[:3], bad])),
             (big, lambda: big.run_grad([torch.ones((9000, 8), device="cuda"), many])),
             (c, lambda: c.run([table[:3], table, bad])),
             (c, lambda: c.run_grad([loss, table[:3], table, bad, loss]))]
    for m, call in calls:
        m._status.fill_(2)
        call()
        with pytest.raises(_lib.FeatGraphError, match="bounded wait"):
            m.device_status()
        assert m.device_status() == 0


@pytest.mark.parametrize("dtype, n", [("float32", 40), ("bfloat16", 40), ("float16", 9000)])
def test_gradient_call_reports_a_label_out_of_range(dtype, n):
    # both ways in which the samples' arrays are made: beside the packing, and (many) by themselves
    feat, weight, labels, dloss = t.xent_inputs(n, 30, 16, dtype, 3)
    m = t.xent_module(feat, weight, labels)
    lse = m.run([feat, weight, labels])[1]
    m.run_grad([dloss, feat, weight, labels, lse])
    assert m.device_status() == 0                        # ignore_index is in range
    for wrong in (30, -1):
        labels[7] = wrong
        m.run_grad([dloss, feat, weight, labels, lse])
        with pytest.raises(_lib.FeatGraphError, match="out of range"):
            m.device_status()


# --------------------------------------- 16 bits: minus infinity in table rows --
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("n, v, d", [(40, 300, 16), (300, 90, 72), (70, 500, 320)])
def test_16_bit_minus_infinity_leaves_the_tables_gradient_alone(dtype, n, v, d):
    # ignored rows, and those behind the last one, meet the infinity as zeros
    feat, weight, labels, dloss = t.xent_inputs(n, v, d, dtype, 9)
    feat[:, 0] = 1.0
    gone = [5, v - 1]
    for row in gone:
        labels[labels == row] = 6
    labels[3] = -100
    kept = [i for i in range(v) if i not in gone]
    place = torch.zeros(v, dtype=torch.int64, device="cuda")
    place[kept] = torch.arange(len(kept), device="cuda")
    small = torch.where(labels == -100, labels, place[labels.clamp(min=0)])
    want = t.xent_reference(feat, weight[kept], small, 1.0, -100, dloss)
    weight[5, 0] = weight[v - 1, 0] = -math.inf
    got = run(t.xent_module(feat, weight, labels), feat, weight, labels, dloss)
    t.check(got["loss"], *want["loss"], torch.float32)
    assert not got["weight_grad"][gone].any()
    t.check(got["weight_grad"][kept], *want["weight_grad"], feat.dtype)
    value, bound = want["feat_grad"]
    t.check(got["feat_grad"][:, 1:], value[:, 1:], bound[:, 1:], feat.dtype)


# ---------------------------------------------------------------- the whole step --
def test_vertex_prediction_takes_arrays_of_the_framework():
    from helpers import random_csr
    from featgraph_b200.pipeline import VertexPrediction
    v, f, n, cols = 120, 16, 50, 90
    step = VertexPrediction(random_csr(n, cols, 0.1, seed=4), v, f, max_norm=0.2)
    g = t.gen(8)
    table = torch.randn((v, f), generator=g, device="cuda")
    ids = torch.randint(v, (cols,), generator=g, device="cuda")
    labels = torch.randint(v, (n,), generator=g, device="cuda")
    labels[::5] = -100

    def copy(out):
        loss, norm, grad = out
        return [x.torch.clone() if isinstance(x, nd.NDArray) else x.clone() for x in (loss, norm, grad)]
    want = copy(step.run(table, ids, labels))
    got = copy(step.run(nd.NDArray(table), nd.NDArray(ids), nd.NDArray(labels)))
    assert all(torch.equal(a, b) for a, b in zip(want, got))


# ---------------------------------------------------------- outputs as inputs --
def test_modules_refuse_their_outputs_as_inputs():
    table = torch.randn((6, 8), device="cuda")
    ids = torch.tensor([5, 0, 3, 3, 1, 2], device="cuda")
    e = module.EmbeddingLookupcuda()
    e.build(t.like(table, ids), {"with_grad": True}, {})
    out = e.run([table, ids])
    with pytest.raises(_lib.FeatGraphError, match="shares memory"):
        e.run([out, ids])
    with pytest.raises(_lib.FeatGraphError, match="shares memory"):
        e.run_grad([e.grad_tvm, ids])
    # two parts of one storage are two arrays
    both = torch.ones((12, 8), device="cuda")
    assert e.run_grad([both[:6], ids], accumulate_into=both[6:]) is not None
    assert torch.equal(both[:6], torch.ones((6, 8), device="cuda"))
    assert both[6:, 0].tolist() == [2, 2, 2, 3, 1, 2]
    k = module.GradientClipcuda()
    grads = [torch.ones(50, device="cuda"), torch.full((50,), 2.0, device="cuda")]
    k.build(t.like(*grads), {"max_norm": 1.0}, {})
    _, clipped = k.run(grads)
    with pytest.raises(_lib.FeatGraphError, match="shares memory"):
        k.run([clipped[1], clipped[0]])
    once = [x.torch.clone() for x in clipped]
    _, again = k.run(clipped)                            # each its own: clipped once more
    assert all(torch.allclose(a, b.torch) for a, b in zip(once, again))


def test_a_device_that_is_not_there_leaves_no_error_behind():
    lib = _lib.load()
    table = torch.randn((6, 8), device="cuda")
    ids = torch.tensor([5, 0, 3], device="cuda")
    out = torch.empty((3, 8), device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()

    def call(device):
        return lib.fg_embedding_lookup(table.data_ptr(), 0, 8, 6, ids.data_ptr(), 1, 3, 8, 1.0,
                                       out.data_ptr(), 8, status.data_ptr(), device, None)
    assert call(99) == 2 and "ordinal" in lib.fg_last_error_string().decode()
    assert call(0) == 0
    torch.cuda.synchronize()
    assert torch.equal(out, table[ids])


# --------------------------------- the table's gradient of more ids than one launch takes --
# 8193 ids and more are sorted; runs of more than 64 rows are cut into windows, those of more than
# 32 parts joined by a whole CTA (60 000 ids of three vertices).
MANY = [(8193, 300, 12), (9001, 97, 20), (30000, 11, 33), (60000, 3, 72)]


@pytest.mark.parametrize("dtype", sorted(t.TYPES))
@pytest.mark.parametrize("index", ["int32", "int64"])
@pytest.mark.parametrize("n, v, f", MANY)
def test_sorted_gradient_padding_accumulate_and_strides(dtype, index, n, v, f):
    g = t.gen(n)
    ids = t.make_ids("skewed", n, v, g).to(getattr(torch, index))
    wide = torch.randn((n, f + 30), generator=g, device="cuda").to(t.TYPES[dtype])
    dy = wide[:, 10:10 + f]
    often = int(torch.bincount(ids.long()).argmax())
    for padding in (None, often, v - 1):
        m = module.EmbeddingLookupcuda()
        m.build([te.placeholder((v, f), dtype)] + t.like(ids),
                {"scale": 0.5, "padding_idx": padding, "with_grad": True}, {})
        m.grad_tvm.torch.fill_(math.nan)
        got = m.run_grad([dy, ids]).torch
        t.check(got, *t.grad_reference(dy, ids, v, 0.5, padding), dy.dtype)
        before = torch.randn((v, f), generator=g, device="cuda").to(t.TYPES[dtype])
        into = before.clone()
        assert m.run_grad([dy, ids], accumulate_into=into) is into
        t.check(into, *t.grad_reference(dy, ids, v, 0.5, padding, before), dy.dtype)
        if padding is not None:
            assert not got[padding].any() and torch.equal(into[padding], before[padding])
        again = before.clone()
        m.run_grad([dy, ids], accumulate_into=again)
        assert torch.equal(again, into) and m.device_status() == 0


@pytest.mark.parametrize("index", ["int32", "int64"])
@pytest.mark.parametrize("n, v, f", MANY)
@pytest.mark.parametrize("wrong", [1, 63, 64, 700, 5000])
def test_sorted_gradient_of_ids_out_of_range(index, n, v, f, wrong):
    g = t.gen(n + wrong)
    ids = t.make_ids("skewed", n, v, g).to(getattr(torch, index))
    dy = torch.randn((n, f), generator=g, device="cuda")
    at = torch.randperm(n, generator=g, device="cuda")[:wrong]
    values = torch.tensor([v, -1, 2 ** 31 - 1, -2 ** 31], device="cuda")
    bad = ids.clone()
    bad[at] = values[torch.arange(wrong, device="cuda") % 4].to(bad.dtype)
    dy[at] = math.nan                                  # and nothing of theirs is added
    m = module.EmbeddingLookupcuda()
    m.build([te.placeholder((v, f), "float32")] + t.like(ids), {"with_grad": True}, {})
    keep = torch.ones(n, dtype=torch.bool, device="cuda")
    keep[at] = False
    want, bound = t.grad_reference(dy[keep], ids[keep], v, 1.0)
    t.check(m.run_grad([dy, bad]).torch, want, bound, torch.float32)
    with pytest.raises(_lib.FeatGraphError, match="out of range"):
        m.device_status()
    before = torch.randn((v, f), generator=g, device="cuda")
    into = before.clone()
    m.run_grad([dy, bad], accumulate_into=into)
    t.check(into, *t.grad_reference(dy[keep], ids[keep], v, 1.0, None, before), torch.float32)


@pytest.mark.parametrize("dtype", sorted(t.TYPES))
@pytest.mark.parametrize("n, v, d", [(20000, 41, 40), (40000, 300, 24), (140000, 41, 16)])
def test_cross_entropy_of_many_samples_and_few_classes(dtype, n, v, d):
    # the table's gradient of a class is a sum over every sample
    feat, weight, labels, dloss = t.xent_inputs(n, v, d, dtype, n)
    t.xent_check(t.xent_module(feat, weight, labels), feat, weight, labels, dloss)


@pytest.mark.parametrize("dtype", sorted(t.TYPES))
def test_cross_entropy_sums_of_one_sign(dtype):
    # Nothing cancels in the gradients' sums, so that what the tensor cores cut adds up: features
    # and weights of one sign.  At most 8192 additions go into one accumulator, each cut by at most
    # 2^-23 of the sum in the worst case (the bound of xent_reference counts every term so).
    feat, weight, labels, dloss = t.xent_inputs(30000, 70, 32, dtype, 5, spread=0.5)
    feat, weight = feat.abs(), weight.abs()
    t.xent_check(t.xent_module(feat, weight, labels), feat, weight, labels, dloss)


@pytest.mark.parametrize("dtype", sorted(t.TYPES))
@pytest.mark.parametrize("scale", [3e38, -3e38])
def test_the_largest_scales_leave_zero_logits_zero(dtype, scale):
    # |scale| log2(e) is beyond float32
    feat = torch.zeros((40, 16), device="cuda", dtype=t.TYPES[dtype])
    weight = torch.randn((300, 16), device="cuda").to(feat.dtype)
    labels = torch.arange(40, device="cuda")
    m = t.xent_module(feat, weight, labels, scale=scale)
    loss, lse = m.run([feat, weight, labels])
    want = math.log(300)
    assert (loss.torch - want).abs().max() <= 400 * U and (lse.torch - want).abs().max() <= 400 * U


# --------------------------------------------------------------- graphs and streams --
def test_vertex_prediction_captured_and_on_another_stream():
    from helpers import random_csr
    from featgraph_b200.pipeline import VertexPrediction
    v, f, n, cols = 200, 24, 60, 110
    step = VertexPrediction(random_csr(n, cols, 0.1, seed=6, empty_rows=(2,)), v, f, scale=1.5, max_norm=0.3)

    def inputs(seed):
        g = t.gen(seed)
        labels = torch.randint(v, (n,), generator=g, device="cuda")
        labels[::4] = -100
        return [torch.randn((v, f), generator=g, device="cuda"),
                torch.randint(v, (cols,), generator=g, device="cuda"), labels]

    def values(out):
        return [out[0].clone(), out[1].torch.clone(), out[2].torch.clone()]
    first, second = inputs(1), inputs(2)
    want = [values(step.run(*x)) for x in (first, second)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = values(step.run(*first))
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want[0], got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step.run(*first)
    for x, y in zip(first, second):
        x.copy_(y)
    for _ in range(2):
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(want[1], values(out)))
    assert all(torch.equal(a, b) for a, b in zip(want[1], values(step.run(*second))))


@pytest.mark.parametrize("warm_up_there", [False, True])
def test_a_graph_outlives_the_build_that_it_was_captured_with(warm_up_there):
    feat, weight, labels, dloss = t.xent_inputs(60, 300, 32, "float32", 3)
    m = t.xent_module(feat, weight, labels)
    want = [x.clone() for x in run(m, feat, weight, labels, dloss).values()]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    if warm_up_there:                                  # the module's last stream is the captured one
        with torch.cuda.stream(stream):
            run(m, feat, weight, labels, dloss)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        outs = list(run(m, feat, weight, labels, dloss).values())
    small = [x[:5] for x in (feat, weight, labels, dloss)]
    small[2] = torch.tensor([0, 1, 2, 3, 4], device="cuda")
    m.build(t.like(small[0], small[1], small[2]), {"with_grad": True}, {})
    # what the allocator has left over goes to others now
    others = [torch.full((size,), 7, dtype=torch.uint8, device="cuda")
              for size in (512, 4096, 40000, 1 << 18, 1 << 20) for _ in range(40)]
    for x in outs:
        x.zero_()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(want, outs))
    assert all(bool((x == 7).all()) for x in others)
    t.check(run(m, *small)["loss"], *t.xent_reference(*small[:3], 1.0, -100)["loss"], torch.float32)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_a_table_read_where_it_lies_takes_no_workspace(dtype):
    n, v, d = 40, 5000, 64
    base = torch.zeros((v + 1) * (d + 8), dtype=t.TYPES[dtype], device="cuda")
    feat, weight, labels, dloss = t.xent_inputs(n, v, d, dtype, 8)
    m = t.xent_module(feat, weight, labels)
    assert m._workspace_size < weight.numel() * 2
    want = [x.clone() for x in run(m, feat, weight, labels, dloss).values()]
    odd = base[1:1 + v * d].view(v, d)                 # off the 16-byte boundaries
    apart = base[:v * (d + 1)].view(v, d + 1)[:, :d]
    for place in (odd, apart, weight):
        if place is not weight:
            place.copy_(weight)
        got = list(run(m, feat, place, labels, dloss).values())
        assert all(torch.equal(a, b) for a, b in zip(want, got))
        assert m._workspace_size > weight.numel() * 2
    assert m.device_status() == 0
    floats = t.xent_module(feat.float(), weight.float(), labels)
    assert floats._workspace_size > weight.numel() * 4


@pytest.mark.parametrize("dtype", sorted(t.TYPES))
def test_a_sample_whose_logits_are_all_minus_infinity(dtype):
    feat, weight, labels, dloss = t.xent_inputs(40, 300, 16, dtype, 9)
    feat[:, 0] = 1.0
    weight[:, 0] = -math.inf
    got = run(t.xent_module(feat, weight, labels), feat, weight, labels, dloss)
    dead = labels == -100
    assert (got["lse"] == -math.inf).all()
    assert got["loss"][~dead].isnan().all() and not got["loss"][dead].any()
