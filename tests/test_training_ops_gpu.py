"""The training operators on the GPU against plain implementations in 64 bits.

Tolerances are worst-case bounds of the arithmetic the operators promise: fp32 (or wider)
sums, u = 2^-24 a rounding, and one rounding to the result's type (half of torch.finfo.eps).
They are evaluated per element from the magnitudes of the terms that were summed.
"""
import math

import numpy as np
import pytest
import torch

from featgraph_b200 import _lib, module, nd, te

pytestmark = pytest.mark.gpu
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
U = 2.0 ** -24


def name(t):
    return str(t.dtype).replace("torch.", "")


def like(*tensors):
    return [te.placeholder(tuple(t.shape), name(t)) for t in tensors]


def half_step(dtype):
    """Largest relative rounding error of the type, and the largest absolute one of its
    subnormal values."""
    f = torch.finfo(dtype)
    return f.eps / 2, f.smallest_normal * f.eps / 2


def check(got, want, bound, dtype):
    """|got - want| <= bound + one rounding of a value within the bound, element by element."""
    rel, tiny = half_step(dtype)
    got, want, bound = got.double(), want.double(), bound.double()
    limit = bound + (want.abs() + bound) * rel + tiny
    over = ~((got - want).abs() <= limit)
    assert not over.any(), "%d of %d off, worst %g times the limit" % (
        int(over.sum()), over.numel(), float(((got - want).abs() / limit).nan_to_num(math.inf).max()))


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---------------------------------------------------------------------- lookup --
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("n, v, f, index", [(0, 5, 8, "int64"), (1, 1, 1, "int32"), (1, 9, 64, "int64"),
                                            (7, 9, 3, "int32"), (33, 9, 8, "int64"), (1000, 77, 33, "int32"),
                                            (513, 300, 100, "int64"), (2049, 4001, 128, "int32"),
                                            (40, 50, 516, "int64")])
def test_lookup(dtype, n, v, f, index):
    g = gen(n + f)
    table = torch.randn((v, f), generator=g, device="cuda").to(TYPES[dtype])
    ids = torch.randint(v, (n,), generator=g, device="cuda").to(getattr(torch, index))
    m = module.EmbeddingLookupcuda()
    m.build(like(table, ids), {"scale": 1.75}, {})
    want = (table.float() * 1.75).to(table.dtype)[ids.long()]
    assert torch.equal(m.run([table, ids]).torch, want)
    out = m.run([nd.NDArray(table), nd.NDArray(ids)])
    assert out is m.out_tvm and torch.equal(out.torch, want)
    assert m.device_status() == 0


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("f, pitch, offset", [(8, 24, 8), (8, 24, 1), (5, 7, 2), (64, 65, 0), (64, 72, 0)])
def test_lookup_of_a_column_slice(dtype, f, pitch, offset):
    base = torch.randn((50, pitch), generator=gen(1), device="cuda").to(TYPES[dtype])
    table = base[:, offset:offset + f]
    ids = torch.tensor([49, 0, 3, 3, 3, 11], dtype=torch.int64, device="cuda")
    m = module.EmbeddingLookupcuda()
    m.build(like(table, ids), {}, {})
    assert torch.equal(m.run([table, ids]).torch, table[ids])


@pytest.mark.parametrize("index", ["int32", "int64"])
def test_lookup_of_an_id_out_of_range(index):
    table = torch.randn((10, 12), device="cuda")
    ids = torch.tensor([3, -1, 10, 9, -2147483648], dtype=getattr(torch, index), device="cuda")
    m = module.EmbeddingLookupcuda()
    m.build(like(table, ids), {"with_grad": True}, {})
    out = m.run([table, ids]).torch
    assert torch.equal(out[[0, 3]], table[[3, 9]]) and out[[1, 2, 4]].isnan().all()
    with pytest.raises(_lib.FeatGraphError, match="out of range"):
        m.device_status()
    assert m.device_status() == 0
    dy = torch.ones((5, 12), device="cuda")
    grad = m.run_grad([dy, ids]).torch
    want = torch.zeros((10, 12), device="cuda")
    want[[3, 9]] = 1
    assert torch.equal(grad, want)
    with pytest.raises(_lib.FeatGraphError, match="out of range"):
        m.device_status()


# ------------------------------------------------------------- lookup: gradient --
def grad_reference(dy, ids, v, scale, padding=None, before=None):
    """The gradient and the bound of its fp32 sums: k terms give (k + 3) u of their magnitudes
    (k - 1 additions of partial sums in any order, at most one more join, the scale)."""
    d = dy.double()
    keep = torch.ones_like(ids, dtype=torch.bool) if padding is None else ids != padding
    ids, d = ids.long()[keep], d[keep]
    want = torch.zeros((v, dy.shape[1]), dtype=torch.float64, device="cuda").index_add_(0, ids, d) * scale
    size = torch.zeros_like(want).index_add_(0, ids, d.abs()) * abs(scale)
    count = torch.zeros(v, dtype=torch.float64, device="cuda").index_add_(0, ids, torch.ones_like(ids, dtype=torch.float64))
    bound = size * (count[:, None] + 3) * U * 1.001
    if before is not None:
        want = want + before.double()
        bound = bound + want.abs() * U
    return want, bound


def make_ids(kind, n, v, g):
    if kind == "flat":
        return torch.randint(v, (n,), generator=g, device="cuda")
    if kind == "same":
        return torch.full((n,), v - 1, device="cuda")
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    return torch.randperm(v, generator=g, device="cuda")[(u ** 4 * v).long()]


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("n, v, f, kind", [
    (1, 1, 1, "flat"), (1, 70001, 12, "flat"), (2, 3, 5, "same"), (31, 4, 8, "flat"), (32, 1, 64, "same"),
    (33, 600, 33, "skewed"), (65, 40, 128, "same"), (4096, 511, 16, "skewed"), (4097, 512, 100, "skewed"),
    (5003, 10007, 100, "skewed"), (20011, 262144, 64, "flat"), (30000, 3, 130, "skewed"),
    (100003, 1000, 24, "skewed"), (66000, 70000, 260, "skewed"), (8192, 5, 40, "flat"), (8192, 7, 136, "same"),
    (8193, 9, 72, "skewed"), (8000, 3, 33, "skewed"), (7000, 1500000, 4, "flat"), (3000, 64, 700, "skewed")])
def test_lookup_grad(dtype, n, v, f, kind):
    g = gen(n + v + f)
    ids = make_ids(kind, n, v, g).to(torch.int32 if n % 2 else torch.int64)
    dy = torch.randn((n, f), generator=g, device="cuda").to(TYPES[dtype])
    m = module.EmbeddingLookupcuda()
    table = te.placeholder((v, f), dtype)
    m.build([table] + like(ids), {"scale": -1.5, "with_grad": True}, {})
    grad = m.run_grad([dy, ids])
    assert grad is m.grad_tvm
    want, bound = grad_reference(dy, ids, v, -1.5)
    check(grad.torch, want, bound, dy.dtype)
    first = grad.torch.clone()
    m.grad_tvm.torch.fill_(math.nan)                  # every element is overwritten
    assert torch.equal(m.run_grad([dy, ids]).torch, first)    # and the bits are the same again


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_lookup_grad_padding_accumulate_and_strides(dtype):
    g = gen(3)
    n, v, f = 3001, 97, 20
    ids = make_ids("skewed", n, v, g)
    wide = torch.randn((n, 50), generator=g, device="cuda").to(TYPES[dtype])
    dy = wide[:, 10:30]
    for padding in (None, int(ids[0]), 0, v - 1):
        m = module.EmbeddingLookupcuda()
        m.build([te.placeholder((v, f), dtype)] + like(ids),
                {"scale": 0.5, "padding_idx": padding, "with_grad": True}, {})
        want, bound = grad_reference(dy, ids, v, 0.5, padding)
        got = m.run_grad([dy, ids]).torch
        check(got, want, bound, dy.dtype)
        if padding is not None:
            assert not got[padding].any()
        before = torch.randn((v, f), generator=g, device="cuda").to(TYPES[dtype])
        into = before.clone()
        assert m.run_grad([dy, ids], accumulate_into=into) is into
        want, bound = grad_reference(dy, ids, v, 0.5, padding, before)
        check(into, want, bound, dy.dtype)
        if padding is not None:
            assert torch.equal(into[padding], before[padding])


@pytest.mark.parametrize("n, distinct", [(8192, 8192), (6000, 500), (8192, 1000)])
def test_lookup_grad_of_ids_that_meet_in_one_slice(n, distinct):
    # vertices that the kernel for few ids deals to one and the same CTA
    high = torch.arange(distinct, device="cuda")
    vertices = high * 128 + ((high ^ (high >> 7) ^ (high >> 14)) & 127)
    g = gen(n)
    ids = vertices[torch.randint(distinct, (n,), generator=g, device="cuda")]
    v = distinct * 128
    dy = torch.randn((n, 4), generator=g, device="cuda")
    m = module.EmbeddingLookupcuda()
    m.build([te.placeholder((v, 4), "float32")] + like(ids), {"with_grad": True}, {})
    want, bound = grad_reference(dy, ids, v, 1.0)
    check(m.run_grad([dy, ids]).torch, want, bound, dy.dtype)


@pytest.mark.parametrize("n", [300, 9000])           # both forms of the gradient
def test_lookup_and_its_gradient_beyond_32_bit_offsets(n):
    v, f = (1 << 25) + 3, 72                            # 2.4e9 elements
    g = gen(n)
    table = torch.zeros((v, f), dtype=torch.float16, device="cuda")
    ids = torch.randint(v - 1000, v, (n,), generator=g, device="cuda")
    ids[:50] = torch.randint(v, (50,), generator=g, device="cuda")
    table[ids] = torch.randn((n, f), generator=g, device="cuda").half()
    m = module.EmbeddingLookupcuda()
    m.build(like(table, ids), {"with_grad": True}, {})
    assert torch.equal(m.run([table, ids]).torch, table[ids])
    dy = torch.randn((n, f), generator=g, device="cuda").half()
    m.grad_tvm.torch.fill_(1.0)
    got = m.run_grad([dy, ids]).torch
    rows, place = torch.unique(ids, return_inverse=True)
    want, bound = grad_reference(dy, place, rows.shape[0], 1.0)
    check(got[rows], want, bound, dy.dtype)
    got[rows] = 0
    assert not got.any()


def test_cross_entropy_beyond_32_bit_offsets():
    n, v, f = 3, (1 << 25) + 3, 72
    g = gen(77)
    feat = torch.randn((n, f), generator=g, device="cuda").half()
    weight = torch.empty((v, f), dtype=torch.float16, device="cuda").normal_(generator=g) * 0.3
    labels = torch.tensor([v - 1, 5, v // 2], device="cuda")
    dloss = torch.tensor([1.0, -2.0, 0.5], device="cuda")
    m = xent_module(feat, weight, labels)
    loss, lse = m.run([feat, weight, labels])
    dh, dw = m.run_grad([dloss, feat, weight, labels, lse])
    # the sum of exponentials by pieces; what the other tests bound per element, here at a few rows
    h = feat.double()
    total = torch.full((n,), -math.inf, dtype=torch.float64, device="cuda")
    for a in range(0, v, 1 << 22):
        total = torch.logaddexp(total, torch.logsumexp(h @ weight[a:a + (1 << 22)].double().T, 1))
    assert ((lse.torch.double() - total).abs() <= 2.0 ** -16).all()
    z = (h * weight[labels].double()).sum(1)
    assert ((loss.torch.double() - (total - z)).abs() <= 2.0 ** -15).all()
    rows = torch.cat([labels, torch.randint(v, (200,), generator=g, device="cuda"),
                      torch.arange(v - 200, v, device="cuda")])
    p = torch.exp(h @ weight[rows].double().T - total[:, None]) * dloss[:, None].double()
    p -= (labels[:, None] == rows[None]) * dloss[:, None].double()
    want = p.T @ h
    bound = (p.abs().T @ h.abs()) * 2.0 ** -10 + 2.0 ** -36 * h.abs().sum(0)
    check(dw.torch[rows], want, bound, torch.float16)


def test_lookup_grad_without_ids():
    m = module.EmbeddingLookupcuda()
    ids = torch.empty(0, dtype=torch.int64, device="cuda")
    m.build([te.placeholder((6, 5), "float32")] + like(ids), {"with_grad": True}, {})
    m.grad_tvm.torch.fill_(7)
    assert not m.run_grad([torch.empty((0, 5), device="cuda"), ids]).torch.any()
    keep = torch.ones((6, 5), device="cuda")
    m.run_grad([torch.empty((0, 5), device="cuda"), ids], accumulate_into=keep)
    assert (keep == 1).all()


def test_lookup_grad_refuses_to_accumulate_into_its_input():
    ids = torch.arange(6, device="cuda")
    dy = torch.ones((6, 4), device="cuda")
    m = module.EmbeddingLookupcuda()
    m.build([te.placeholder((6, 4))] + like(ids), {"with_grad": True}, {})
    with pytest.raises(ValueError, match="share memory"):
        m.run_grad([dy, ids], accumulate_into=dy)


def test_lookup_grad_nan_reaches_only_its_vertex():
    ids = torch.arange(500, device="cuda") % 50
    dy = torch.ones((500, 16), device="cuda")
    dy[7] = math.nan
    m = module.EmbeddingLookupcuda()
    m.build([te.placeholder((50, 16), "float32")] + like(ids), {"with_grad": True, "padding_idx": 9}, {})
    dy[9] = math.inf                                   # a row of the padding id
    got = m.run_grad([dy, ids]).torch
    assert got[7].isnan().all() and not got[9].any()
    rest = [v for v in range(50) if v not in (7, 9)]
    assert (got[rest] == 10).all()


# --------------------------------------------------------------- cross entropy --
def xent_reference(feat, weight, labels, scale, ignore, dloss=None):
    """Losses and gradients in fp64 with worst-case error bounds.

    A logit is a sum of D products in fp32: (D + 8) u of the terms' magnitudes, twice that for
    tensor-core sums that cut instead of round; float32 operands split into two pieces lose
    2^-21 of each product.  exp and log add a few u; the sum of V exponentials V u.  dz is
    rounded to 16 bits (or two pieces, 2^-21) before the products of the gradients, which are
    sums like the logits'."""
    exact32 = feat.dtype == torch.float32
    split = 2.0 ** -21 if exact32 else 0.0
    h, w = feat.double(), weight.double()
    n, d = h.shape
    v = w.shape[0]
    keep = labels != ignore
    z = scale * (h @ w.T)
    ez = abs(scale) * (h.abs() @ w.abs().T) * ((d + 8) * 2 * U + split)
    lse = torch.logsumexp(z, 1)
    elz = ez.amax(1) + (v + 64) * U + lse.abs() * 4 * U
    at = torch.where(keep, labels.long(), 0)[:, None]
    loss = torch.where(keep, lse - z.gather(1, at)[:, 0], 0.0)
    eloss = torch.where(keep, elz + ez.gather(1, at)[:, 0] + loss.abs() * 2 * U, 0.0)
    out = {"loss": (loss, eloss), "lse": (lse, elz)}
    if dloss is None:
        return out
    g = torch.where(keep, dloss.double(), 0.0)[:, None]
    p = torch.exp(z - lse[:, None])
    dz = p.clone()
    dz.scatter_add_(1, at, -torch.ones_like(at, dtype=torch.float64))
    dz = dz * g * scale
    ep = p * (torch.expm1(ez + elz[:, None]) + 16 * U) * (g * scale).abs()
    # fp16 pieces end at 2^-40 of the largest magnitude, |scale| * max |loss_grad|
    ends = abs(scale) * float(g.abs().max()) * 2.0 ** -38
    edz = ep + (dz.abs() + ep) * (2.0 ** -21 if exact32 else half_step(feat.dtype)[0]) + ends
    hk = torch.where(keep[:, None], h, 0.0)
    sums = (2 * U, split)
    out["feat_grad"] = (dz @ w, edz @ w.abs() + (dz.abs() @ w.abs()) * ((v + 8) * sums[0] + sums[1]))
    out["weight_grad"] = (dz.T @ hk, edz.T @ hk.abs() + (dz.abs().T @ hk.abs()) * ((n + 8) * sums[0] + sums[1]))
    out["feat_grad"] = tuple(torch.where(keep[:, None], x, 0.0) for x in out["feat_grad"])
    return out


XENT_SIZES = [(1, 1, 1), (1, 7, 3), (2, 33, 8), (5, 1000, 64), (31, 129, 16), (128, 256, 64),
              (129, 257, 65), (131, 2003, 100), (257, 517, 33), (64, 4097, 128), (300, 10007, 32),
              (1, 20011, 130), (1027, 700, 24), (40, 90, 600), (200, 1500, 192), (150, 700, 256),
              (400, 2600, 260), (97, 3000, 448)]


def xent_inputs(n, v, d, dtype, seed, spread=2.0):
    g = gen(seed)
    feat = torch.randn((n, d), generator=g, device="cuda").to(TYPES[dtype])
    weight = (torch.randn((v, d), generator=g, device="cuda") * spread * d ** -0.5).to(TYPES[dtype])
    labels = torch.randint(v, (n,), generator=g, device="cuda")
    labels[torch.rand(n, generator=g, device="cuda") < 0.2] = -100
    dloss = (torch.rand(n, generator=g, device="cuda") + 0.5) / n
    return feat, weight, labels, dloss


def xent_module(feat, weight, labels, **args):
    m = module.SoftmaxCrossEntropycuda()
    m.build(like(feat, weight, labels), dict({"with_grad": True}, **args), {})
    return m


def xent_check(m, feat, weight, labels, dloss, scale=1.0, ignore=-100):
    want = xent_reference(feat, weight, labels, scale, ignore, dloss)
    loss, lse = m.run([feat, weight, labels])
    dh, dw = m.run_grad([dloss, feat, weight, labels, lse])
    got = {"loss": loss.torch, "lse": lse.torch, "feat_grad": dh.torch, "weight_grad": dw.torch}
    for key, (value, bound) in want.items():
        check(got[key], value, bound, got[key].dtype)
    return got


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("n, v, d", XENT_SIZES)
def test_cross_entropy(dtype, n, v, d):
    feat, weight, labels, dloss = xent_inputs(n, v, d, dtype, n + v + d)
    if n % 2:
        labels = labels.to(torch.int32)
    m = xent_module(feat, weight, labels, scale=0.75)
    got = xent_check(m, feat, weight, labels, dloss, 0.75)
    dead = labels == -100
    assert not got["loss"][dead].any() and not got["feat_grad"][dead].any()
    again = {k: x.clone() for k, x in got.items()}
    for x in got.values():
        x.fill_(math.nan)                              # every element is overwritten
    got = xent_check(m, feat, weight, labels, dloss, 0.75)
    assert all(torch.equal(got[k], again[k]) for k in got)
    assert m.device_status() == 0


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("d, offset, pitch", [(64, 0, 72), (64, 1, 72), (40, 8, 56), (33, 0, 40)])
def test_cross_entropy_of_column_slices(dtype, d, offset, pitch):
    feat, weight, labels, dloss = xent_inputs(70, 333, pitch, dtype, d)
    feat, weight = feat[:, offset:offset + d], weight[:, offset:offset + d]
    xent_check(xent_module(feat, weight, labels), feat, weight, labels, dloss)


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_cross_entropy_ignored_rows_take_no_part(dtype):
    feat, weight, labels, dloss = xent_inputs(150, 400, 48, dtype, 5)
    labels[3:9] = 7                                    # another ignore index than the default
    labels[labels == -100] = 8
    clean = xent_check(xent_module(feat, weight, labels, ignore_index=7), feat, weight, labels,
                       dloss, ignore=7)
    clean = {k: x.clone() for k, x in clean.items()}
    feat[3], feat[4], dloss[5], dloss[3] = math.nan, math.inf, math.nan, math.inf
    m = xent_module(feat, weight, labels, ignore_index=7)
    loss, lse = m.run([feat, weight, labels])
    dh, dw = m.run_grad([dloss, feat, weight, labels, lse])
    assert torch.equal(loss.torch, clean["loss"])
    assert torch.equal(dh.torch, clean["feat_grad"]) and torch.equal(dw.torch, clean["weight_grad"])
    labels.fill_(7)                                    # nothing is left
    loss, lse = m.run([feat, weight, labels])
    dh, dw = m.run_grad([dloss, feat, weight, labels, lse])
    assert not loss.torch.any() and not dh.torch.any() and not dw.torch.any()


def test_cross_entropy_of_a_label_out_of_range():
    feat, weight, labels, dloss = xent_inputs(20, 50, 16, "float32", 6)
    labels[:] = torch.arange(20, device="cuda")
    ok = xent_module(feat, weight, labels)
    loss = ok.run([feat, weight, labels])[0].torch.clone()
    bad = labels.clone()
    bad[4], bad[5] = 50, -1
    m = xent_module(feat, weight, bad)
    got, lse = m.run([feat, weight, bad])
    keep = [i for i in range(20) if i not in (4, 5)]
    assert got.torch[[4, 5]].isnan().all() and torch.equal(got.torch[keep], loss[keep])
    with pytest.raises(_lib.FeatGraphError, match="out of range"):
        m.device_status()
    dh, dw = m.run_grad([dloss, feat, weight, bad, lse])
    assert not dh.torch[[4, 5]].any()
    labels[4] = labels[5] = -100
    lse2 = ok.run([feat, weight, labels])[1]
    dh2, dw2 = ok.run_grad([dloss, feat, weight, labels, lse2])
    assert torch.equal(dh.torch, dh2.torch) and torch.equal(dw.torch, dw2.torch)


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_cross_entropy_far_logits(dtype):
    # logits of a few hundred: exp of an unshifted logit would overflow
    feat, weight, labels, dloss = xent_inputs(90, 700, 64, dtype, 8, spread=60.0)
    xent_check(xent_module(feat, weight, labels), feat, weight, labels, dloss)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("n, v", [(200, 40), (70, 3001)])
@pytest.mark.parametrize("scale", [-0.5, 0.0, 3.0])
def test_cross_entropy_signs(dtype, n, v, scale):
    # negative and zero weights of the losses, negative and zero scales, sizes apart by 2^12
    feat, weight, labels, dloss = xent_inputs(n, v, 72, dtype, 12)
    dloss = dloss * torch.randn(n, generator=gen(13), device="cuda")
    dloss[::9] = 0.0
    dloss[4] *= 4096.0
    xent_check(xent_module(feat, weight, labels, scale=scale), feat, weight, labels, dloss, scale)


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_cross_entropy_one_gradient_alone_and_many_samples(dtype):
    # more samples than the single-CTA preparation takes, few classes: the samples are split
    feat, weight, labels, dloss = xent_inputs(8300, 17, 20, dtype, 14)
    xent_check(xent_module(feat, weight, labels), feat, weight, labels, dloss)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_cross_entropy_minus_infinity_beside_finite_logits(dtype):
    feat, weight, labels, _ = xent_inputs(40, 300, 16, dtype, 9)
    feat[:, 0] = 1.0
    weight[5, 0] = weight[299, 0] = -math.inf          # these vertices never
    labels[labels == 5] = 6
    labels[labels == 299] = 6
    m = xent_module(feat, weight, labels)
    loss, lse = m.run([feat, weight, labels])
    finite = [v for v in range(300) if v not in (5, 299)]
    shift = labels - (labels > 5).to(labels.dtype)
    want = xent_reference(feat, weight[finite], torch.where(labels == -100, labels, shift), 1.0, -100)
    check(loss.torch, *want["loss"], torch.float32)
    check(lse.torch, *want["lse"], torch.float32)


@pytest.mark.parametrize("along", ["random", "gradient"])
def test_cross_entropy_gradient_against_differences(along):
    # f(e) = sum_t g_t loss_t at feat + e dF, weight + e dW; bilinear logits, so the difference
    # quotient misses f'(0) by at most e^2/6 sup|f'''| plus the losses' own error over e
    feat, weight, labels, dloss = xent_inputs(60, 500, 32, "float32", 10)
    g = gen(11)
    df = torch.randn(feat.shape, generator=g, device="cuda") * 0.1
    dw = torch.randn(weight.shape, generator=g, device="cuda") * 0.02
    m = xent_module(feat, weight, labels)
    _, lse = m.run([feat, weight, labels])
    gf, gw = m.run_grad([dloss, feat, weight, labels, lse])
    if along == "gradient":                            # the direction in which it changes most
        df = gf.torch / gf.torch.abs().max() * 0.3
        dw = gw.torch / gw.torch.abs().max() * 0.05
    slope = float((gf.torch.double() * df).sum() + (gw.torch.double() * dw).sum())
    e, values, noise = 2.0 ** -5, [], 0.0
    for s in (e, -e):
        a, b = feat + s * df, weight + s * dw
        ref = xent_reference(a, b, labels, 1.0, -100)
        noise += float((ref["loss"][1] * dloss).sum())
        values.append(float((m.run([a, b, labels])[0].torch.double() * dloss).sum()))
    # z(e) = z0 + e z1 + e^2 z2: f''' of a log-sum-exp is a third cumulant of z' plus three
    # times a covariance of z' and z''; both moments are at most powers of the ranges
    f64, w64 = feat.double(), weight.double()
    z2 = df.double() @ dw.double().T
    z1 = f64 @ dw.double().T + df.double() @ w64.T
    r1 = (z1.amax(1) - z1.amin(1)) + 2 * e * (z2.amax(1) - z2.amin(1))
    r2 = 2 * (z2.amax(1) - z2.amin(1))
    third = float(((r1 ** 3 + 3 * r1 * r2) * dloss).sum())
    # slope's own error: the gradients' bounds against |df|, |dw|
    want = xent_reference(feat, weight, labels, 1.0, -100, dloss)
    own = float((want["feat_grad"][1] * df.abs()).sum() + (want["weight_grad"][1] * dw.abs()).sum())
    quotient = (values[0] - values[1]) / (2 * e)
    assert abs(quotient - slope) <= e * e / 6 * third + noise / (2 * e) + own
    if along == "gradient":                            # where the bound is far below the slope
        assert slope > 3 * (e * e / 6 * third + noise / (2 * e) + own)


def test_feature_lengths_in_any_order_in_a_fresh_process():
    # the kernels' shared memory depends on the feature length: a shorter one in between must not
    # take from a longer one what it was allowed before
    import os
    import subprocess
    import sys
    code = """
import sys, torch
sys.path[:0] = [%r, %r]
import test_training_ops_gpu as t
for dtype in sorted(t.TYPES):
    for d in (128, 16, 128, 256, 40, 256, 70, 500, 20, 500):
        feat, weight, labels, dloss = t.xent_inputs(40, 300, d, dtype, d)
        t.xent_check(t.xent_module(feat, weight, labels), feat, weight, labels, dloss)
""" % (os.path.dirname(os.path.abspath(__file__)),
       os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_cross_entropy_of_nothing():
    m = module.SoftmaxCrossEntropycuda()
    feat = torch.empty((0, 8), device="cuda")
    weight = torch.randn((30, 8), device="cuda")
    labels = torch.empty(0, dtype=torch.int64, device="cuda")
    m.build(like(feat, weight, labels), {"with_grad": True}, {})
    m.weight_grad_tvm.torch.fill_(3)
    loss, lse = m.run([feat, weight, labels])
    dh, dw = m.run_grad([loss, feat, weight, labels, lse])
    assert loss.shape == (0,) and dh.shape == (0, 8) and not dw.torch.any()


# ------------------------------------------------------------------------- clip --
CLIP_SHAPES = [[(1,)], [(5,), (0,), (3, 4)], [(100, 33), (33,)], [(8192,), (8193,), (1,)],
               [(300, 1001), (64, 64), (7,)], [(3,)] * 70, [(11, 5)] * 1030]


@pytest.mark.parametrize("norm_type", [2, math.inf])
@pytest.mark.parametrize("dtype", sorted(TYPES) + ["mixed"])
@pytest.mark.parametrize("shapes", CLIP_SHAPES, ids=lambda s: "%dx%s" % (len(s), s[0]))
@pytest.mark.parametrize("ratio", [0.3, 3.0])
def test_clip(norm_type, dtype, shapes, ratio):
    g = gen(len(shapes))
    order = sorted(TYPES)
    grads = [torch.randn(s, generator=g, device="cuda").to(TYPES[order[k % 3] if dtype == "mixed" else dtype])
             for k, s in enumerate(shapes)]
    flat = torch.cat([x.double().flatten() for x in grads])
    true = float(torch.linalg.vector_norm(flat, norm_type))
    m = module.GradientClipcuda()
    args = {"max_norm": ratio * true, "norm_type": norm_type}
    m.build(like(*grads), args, {})
    norm, clipped = m.run(grads)
    # squares of eight in fp32 before fp64: 8 u of the sum, half of it after the root, and the
    # result's own rounding; the factor and the product are rounded once more each
    assert abs(float(norm.torch) - true) <= true * 6 * U
    share = min(1.0, ratio * true / (true + 1e-6))
    for x, y in zip(grads, clipped):
        want = x.double() * share
        check(y.torch, want, want.abs() * 8 * U, x.dtype)
    if ratio > 1:
        assert all(torch.equal(x, y.torch) for x, y in zip(grads, clipped))
    keep = [x.clone() for x in grads]
    p = module.GradientClipcuda()
    p.build(like(*grads), dict(args, in_place=True), {})
    norm2, same = p.run(keep)
    assert all(a is b for a, b in zip(same, keep))
    assert torch.equal(norm2.torch, norm.torch)
    assert all(torch.equal(a, b.torch) for a, b in zip(keep, clipped))


def test_clip_of_odd_addresses_and_ranges():
    base = torch.randn(10001, generator=gen(4), device="cuda")
    grads = [base[1:4000], base[4001:9000], base[9001:9002]]          # 4-byte alignment only
    m = module.GradientClipcuda()
    m.build(like(*grads), {"max_norm": 1.0}, {})
    norm, clipped = m.run(grads)
    true = float(torch.linalg.vector_norm(torch.cat(grads).double()))
    assert abs(float(norm.torch) - true) <= true * 6 * U
    # squares beyond and below the range of fp32
    for size in (1e30, 1e-30):
        x = [torch.full((777,), size, device="cuda"), torch.full((5,), -size, device="cuda")]
        m = module.GradientClipcuda()
        m.build(like(*x), {"max_norm": size, "eps": 0.0}, {})
        norm, clipped = m.run(x)
        want = size * math.sqrt(782)
        assert abs(float(norm.torch) - want) <= want * 8 * U
        check(clipped[1].torch, x[1].double() / math.sqrt(782),
              x[1].double().abs() / math.sqrt(782) * 12 * U, torch.float32)


@pytest.mark.parametrize("norm_type", [2, math.inf])
def test_clip_of_nan_and_infinity(norm_type):
    for bad, out in ((math.nan, math.nan), (math.inf, 0.0)):
        x = [torch.ones(1000, device="cuda"), torch.ones(33, device="cuda").bfloat16()]
        x[0][777] = bad
        m = module.GradientClipcuda()
        m.build(like(*x), {"max_norm": 1.0, "norm_type": norm_type}, {})
        norm, clipped = m.run(x)
        assert math.isnan(float(norm.torch)) == math.isnan(bad)
        assert torch.equal(clipped[1].torch.nan_to_num(9), torch.full_like(x[1], out).nan_to_num(9))
        free = module.GradientClipcuda()                 # without a bound nothing is scaled
        free.build(like(*x), {"norm_type": norm_type}, {})
        assert torch.equal(free.run(x)[1][1].torch, x[1])


def test_clip_of_nothing():
    m = module.GradientClipcuda()
    m.build([], {"max_norm": 1.0}, {})
    norm, clipped = m.run([])
    assert float(norm.torch) == 0 and clipped == []


def test_clip_refuses_shared_memory_in_place():
    x = torch.ones(100, device="cuda")
    m = module.GradientClipcuda()
    m.build(like(x[:60], x[50:]), {"max_norm": 1.0, "in_place": True}, {})
    with pytest.raises(ValueError, match="share memory"):
        m.run([x[:60], x[50:]])
    m.run([x[:60], x[50:].clone()])


# ------------------------------------------------- refusals, streams and capture --
def test_module_refusals():
    table = torch.randn((10, 8), device="cuda")
    ids = torch.zeros(4, dtype=torch.int64, device="cuda")
    m = module.EmbeddingLookupcuda()
    with pytest.raises(RuntimeError, match="build"):
        m.run([table, ids])
    m.build(like(table, ids), {}, {})
    with pytest.raises(RuntimeError, match="with_grad"):
        m.run_grad([torch.zeros((4, 8), device="cuda"), ids])
    with pytest.raises(ValueError, match="exactly 2"):
        m.run([table])
    with pytest.raises(TypeError, match="dtype"):
        m.run([table.half(), ids])
    with pytest.raises(TypeError, match="dtype"):
        m.run([table, ids.int()])
    with pytest.raises(ValueError, match="shape"):
        m.run([table[:9], ids])
    with pytest.raises(ValueError, match="lives on"):
        m.run([table.cpu(), ids])
    with pytest.raises(TypeError, match="NDArray"):
        m.run([table.cpu().numpy(), ids])
    with pytest.raises(ValueError, match="strides"):
        m.run([torch.randn((8, 10), device="cuda").T, ids])
    with pytest.raises(ValueError, match="strides"):
        m.run([torch.randn((1, 8), device="cuda").expand(10, 8), ids])
    with pytest.raises(ValueError, match="contiguous"):
        m.run([table, torch.zeros(8, dtype=torch.int64, device="cuda")[::2]])
    c = module.SoftmaxCrossEntropycuda()
    c.build(like(table[:4], table, ids), {}, {})
    with pytest.raises(RuntimeError, match="with_grad"):
        c.run_grad([torch.zeros(4, device="cuda"), table[:4], table, ids, torch.zeros(4, device="cuda")])
    with pytest.raises(ValueError, match="exactly 3"):
        c.run([table[:4], table])


def _operators(seed):
    """One built module of each kind with its inputs: (call, outputs) pairs."""
    g = gen(seed)
    ids = make_ids("skewed", 3000, 200, g)
    table = torch.randn((200, 48), generator=g, device="cuda")
    dy = torch.randn((3000, 48), generator=g, device="cuda")
    e = module.EmbeddingLookupcuda()
    e.build(like(table, ids), {"with_grad": True}, {})
    feat, weight, labels, dloss = xent_inputs(90, 300, 48, "bfloat16", seed)
    c = xent_module(feat, weight, labels)
    k = module.GradientClipcuda()
    k.build(like(table, dy), {"max_norm": 1.0}, {})

    def call():
        out = [e.run([table, ids]).torch, e.run_grad([dy, ids]).torch]
        loss, lse = c.run([feat, weight, labels])
        out += [loss.torch, lse.torch]
        out += [x.torch for x in c.run_grad([dloss, feat, weight, labels, lse])]
        norm, clipped = k.run([table, dy])
        return out + [norm.torch] + [x.torch for x in clipped]
    inputs = [table, ids, dy, feat, weight, labels, dloss]
    return call, inputs


def test_other_streams_and_captured_graphs_give_the_same_bits():
    call, inputs = _operators(21)
    want = [x.clone() for x in call()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [x.clone() for x in call()]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = call()
    other, fresh = _operators(22)
    want2 = [x.clone() for x in other()]
    for x, y in zip(inputs, fresh):
        x.copy_(y)                                     # new inputs in the captured places
    for _ in range(3):
        for x in outs:
            x.zero_()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(want2, outs))


def test_modules_side_by_side_on_streams_and_threads():
    # each host thread with modules and a stream of its own; the tensor-core kernels of the
    # others hold the machine in between
    import threading
    cases = []
    for seed in (31, 32, 33):
        call, _ = _operators(seed)
        cases.append((call, [x.clone() for x in call()], torch.cuda.Stream(), []))
    torch.cuda.synchronize()

    def work(call, want, stream, wrong):
        with torch.cuda.stream(stream):
            for _ in range(20):
                got = call()
                wrong.extend(not torch.equal(a, b) for a, b in zip(want, got))
    threads = [threading.Thread(target=work, args=c) for c in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert all(len(c[3]) == 20 * len(c[1]) and not any(c[3]) for c in cases)


@pytest.mark.parametrize("size", [1e-30, 1e-4, 1e4, 1e15])
def test_cross_entropy_float32_operands_of_any_size(size):
    # the fp16 pieces are relative to the operands' largest values; scale brings the logits back
    feat, weight, labels, dloss = xent_inputs(50, 400, 40, "float32", 15)
    xent_check(xent_module(feat, weight * size, labels, scale=1.0 / size), feat, weight * size,
               labels, dloss, 1.0 / size)
    xent_check(xent_module(feat * size, weight, labels, scale=1.0 / size), feat * size, weight,
               labels, dloss, 1.0 / size)


def test_the_rest_of_the_module_interface():
    table = torch.randn((40, 8), device="cuda")
    ids = torch.arange(20, device="cuda")
    e, c, k = module.EmbeddingLookupcuda(), module.SoftmaxCrossEntropycuda(), module.GradientClipcuda()
    e.build(like(table, ids), {}, {})
    c.build(like(table[:20], table, ids), {}, {})
    k.build(like(table), {"max_norm": 1.0, "in_place": True}, {})
    for m, inputs in ((e, [table, ids]), (c, [table[:20], table, ids]), (k, [table.clone()])):
        assert m.measure_average_time(inputs, 3) > 0
        assert m.target == "cuda" and repr(m.ctx) == "gpu(0)" and m.device_status() == 0
    text = c.lower_to_ir(like(table[:20], table, ids), {"with_grad": True}, {})
    assert "softmax_cross_entropy" in text and "workspace" in text
    with pytest.raises(RuntimeError, match="build"):
        module.GradientClipcuda().run([table])
    assert module.EmbeddingLookupcuda().device_status() == 0      # nothing built, nothing wrong


def test_build_again_with_other_shapes():
    m = module.SoftmaxCrossEntropycuda()
    for n, v, d in ((5, 40, 8), (200, 30, 64), (3, 1000, 16)):
        feat, weight, labels, dloss = xent_inputs(n, v, d, "float32", n)
        m.build(like(feat, weight, labels), {"with_grad": True}, {})
        xent_check(m, feat, weight, labels, dloss)


def test_a_training_step_of_a_layer():
    """Lookup -> SpMM -> loss over all vertices with tied weights -> gradients back through the
    SpMM of the transposed adjacency and the lookup -> clip; every stage against 64 bits of its
    own inputs."""
    from helpers import random_csr
    v, f, n = 400, 32, 150
    adj = random_csr(n, 600, 0.05, seed=9, empty_rows=(3,))
    g = gen(30)
    table = torch.randn((v, f), generator=g, device="cuda") * 0.3
    ids = make_ids("skewed", 600, v, g)
    labels = torch.randint(v, (n,), generator=g, device="cuda")
    labels[3] = -100
    dloss = torch.full((n,), 1.0 / n, device="cuda")
    dense = torch.from_numpy(adj.toarray()).cuda().double()

    look = module.EmbeddingLookupcuda()
    look.build([te.placeholder((v, f)), te.placeholder((600,), "int64")],
               {"scale": f ** 0.5, "with_grad": True}, {})
    spmm, back = module.VanillaSpMMcuda(adj), module.VanillaSpMMcuda(adj.T.tocsr())
    spmm.build([te.placeholder((600, f))], {}, {})
    back.build([te.placeholder((n, f))], {}, {})
    loss_op = module.SoftmaxCrossEntropycuda()
    loss_op.build([te.placeholder((n, f)), te.placeholder((v, f)), te.placeholder((n,), "int64")],
                  {"with_grad": True}, {})
    clip = module.GradientClipcuda()
    clip.build([te.placeholder((v, f))], {"max_norm": 0.1}, {})

    x = look.run([table, ids])
    assert torch.equal(x.torch, table[ids] * np.float32(f ** 0.5))
    y = spmm.run([x])
    def spmm_bound(a, b):
        return (a.abs() @ b.double().abs()) * (a.shape[1] + 2) * U
    check(y.torch, dense @ x.torch.double(), spmm_bound(dense, x.torch), torch.float32)
    loss, lse = loss_op.run([y, table, labels])
    want = xent_reference(y.torch, table, labels, 1.0, -100, dloss)
    check(loss.torch, *want["loss"], torch.float32)
    dy, dtable = loss_op.run_grad([dloss, y, table, labels, lse])
    check(dy.torch, *want["feat_grad"], torch.float32)
    check(dtable.torch, *want["weight_grad"], torch.float32)
    dx = back.run([dy])
    check(dx.torch, dense.T @ dy.torch.double(), spmm_bound(dense.T, dy.torch), torch.float32)
    before = dtable.torch.clone()
    total = look.run_grad([dx, ids], accumulate_into=dtable)
    assert total is dtable
    check(dtable.torch, *grad_reference(dx.torch, ids, v, f ** 0.5, None, before), torch.float32)
    norm, (out,) = clip.run([dtable])
    true = float(dtable.torch.double().norm())
    assert abs(float(norm.torch) - true) <= true * 6 * U and true > 0.1
    share = 0.1 / (true + 1e-6)
    check(out.torch, dtable.torch.double() * share, dtable.torch.double().abs() * share * 8 * U,
          torch.float32)
    for m in (look, loss_op, spmm, back):
        assert m.device_status() == 0


@pytest.mark.parametrize("index", ["int32", "int64"])
def test_vertex_prediction_is_its_parts_and_follows_new_inputs(index):
    # the composed step against 64-bit autograd of the formula: forward and backward are chains
    # of sums whose terms' magnitudes the same formula gives with absolute values
    from helpers import random_csr
    from featgraph_b200.pipeline import VertexPrediction
    v, f, n, cols = 300, 24, 90, 400
    adj = random_csr(n, cols, 0.03, seed=4, empty_rows=(5, 6))
    dense = torch.from_numpy(adj.toarray()).cuda().double()
    step = VertexPrediction(adj, v, f, scale=2.0, scale_out=0.3, max_norm=0.2, index_dtype=index)
    for seed in (1, 2):
        g = gen(seed)
        table = torch.randn((v, f), generator=g, device="cuda") * 0.3
        ids = make_ids("skewed", cols, v, g).to(getattr(torch, index))
        labels = torch.randint(v, (n,), generator=g, device="cuda").to(getattr(torch, index))
        labels[::7] = -100
        loss, norm, grad = step.run(table, ids, labels)
        t = table.double().requires_grad_()
        z = 0.3 * (dense @ (2.0 * t[ids.long()])) @ t.T
        want = torch.nn.functional.cross_entropy(z, labels.long(), ignore_index=-100)
        want.backward()
        want = float(want.detach())
        true = float(t.grad.norm())
        # relative errors add up along the chain: lookup 1, SpMM degree (< 60), logits 2 (f + 8),
        # softmax v + 64, two products 2 (v + 8), back through the SpMM 60 and the lookup 60;
        # against a gradient that cancels by less than 20 in norm: 1500 u * 20
        tol = 1500 * U * 20
        assert abs(float(loss) - want) <= tol * abs(want)
        assert abs(float(norm.torch) - true) <= tol * true
        scaled = t.grad * (0.2 / (true + 1e-6))
        assert float((grad.torch.double() - scaled).norm()) <= tol * float(scaled.norm())
    assert step.device_status() == 0
