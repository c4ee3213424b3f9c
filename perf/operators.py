"""The training operators that stand next to the SpMM and the SDDMM, as measurable cases.

Three operators: the vertex embedding lookup with its gradient, the softmax cross entropy over
all vertices (or classes) with its gradients, and the global gradient norm with clipping.
``run`` computes a case in its plain form (elementary torch operations in 32 bits, rounded
once at the end) or, with ``own`` set, through this repository's modules.
"""
import math

import torch

own = False

VERTICES = 232965          # the vertex count of the repository's benchmark graph
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
INDEX = {"int32": torch.int32, "int64": torch.int64}
IGNORE = -100
SKEW = 4.0                 # ids are floor(V * u**SKEW) through a permutation: a power law


def listed():
    return [
        # one vertex served online: the call's latency
        dict(name="lookup_one", op="lookup", n=1, vertices=VERTICES, feat=64, dtype="float32",
             index="int64", scale=1.0, seeds="skewed"),
        # the input features of a sampled neighbourhood of a large mini-batch
        dict(name="lookup_batch", op="lookup", n=1048576, vertices=VERTICES, feat=128,
             dtype="bfloat16", index="int32", scale=11.25, seeds="skewed"),
        # a small ragged batch, odd feature length, over the vertices of a small graph
        dict(name="lookup_grad_ragged", op="lookup_grad", n=5003, vertices=10007, feat=100,
             dtype="float32", index="int64", scale=10.0, seeds="skewed"),
        # the gradient of the large mini-batch: popular vertices repeat tens of thousands of times
        dict(name="lookup_grad_batch", op="lookup_grad", n=1048576, vertices=VERTICES, feat=128,
             dtype="bfloat16", index="int32", scale=11.25, seeds="skewed"),
        # the same in the framework's own type, every vertex about equally often
        dict(name="lookup_grad_flat", op="lookup_grad", n=600011, vertices=VERTICES, feat=64,
             dtype="float32", index="int64", scale=1.0, seeds="flat"),
        # one query scored against every vertex
        dict(name="xent_one", op="xent", n=1, vertices=VERTICES, feat=128, dtype="bfloat16",
             index="int64", scale=1.0, ignored=0.0),
        # evaluation of a large batch against every vertex
        dict(name="xent_batch", op="xent", n=4096, vertices=VERTICES, feat=256,
             dtype="bfloat16", index="int64", scale=1.0, ignored=0.05),
        # a training step of a small ragged batch, odd sizes throughout
        dict(name="xent_train_ragged", op="xent_train", n=131, vertices=10007, feat=100,
             dtype="float16", index="int32", scale=0.5, ignored=0.3),
        # a training step against every vertex
        dict(name="xent_train_batch", op="xent_train", n=4096, vertices=VERTICES, feat=256,
             dtype="bfloat16", index="int64", scale=1.0, ignored=0.05),
        # a training step in the framework's own type over a middling graph
        dict(name="xent_train_f32", op="xent_train", n=2048, vertices=50021, feat=128,
             dtype="float32", index="int64", scale=1.0, ignored=0.05),
        # the gradients of one small layer: weight and bias
        dict(name="clip_layer", op="clip", tensors=2, largest=16384, dtype="float32",
             norm="l2", ratio=0.25),
        # a table of vertex embeddings and the layers above it
        dict(name="clip_model", op="clip", tensors=48, largest=VERTICES * 128,
             dtype="float32", norm="l2", ratio=0.25),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["lookup", "lookup_grad", "xent", "xent_train", "clip"])
    dtype = rng.choice(sorted(TYPES))
    if op == "clip":
        return dict(op=op, tensors=_log(rng, 1, 60), largest=_log(rng, 5, VERTICES * 64),
                    dtype=dtype, norm=rng.choice(["l2", "l2", "max"]),
                    ratio=rng.choice([0.1, 0.5, 2.0]))
    index = rng.choice(sorted(INDEX))
    scale = round(rng.uniform(0.25, 4.0), 3)
    if op in ("lookup", "lookup_grad"):
        return dict(op=op, n=_log(rng, 1, 500000), vertices=_log(rng, 10, VERTICES),
                    feat=_log(rng, 1, 200), dtype=dtype, index=index, scale=scale,
                    seeds=rng.choice(["skewed", "flat"]))
    big = 32 if dtype == "float32" else 256
    return dict(op=op, n=_log(rng, 1, 2000), vertices=_log(rng, 10, VERTICES // 2),
                feat=_log(rng, 8, big), dtype=dtype, index=index, scale=min(scale, 1.5),
                ignored=rng.choice([0.0, 0.2]))


def _sizes(case):
    """Element counts of a model's gradients: one table, matrices of falling size, biases."""
    k = case["tensors"]
    return [max(1, int(case["largest"] / (1.0 if i == 0 else 4.0 * (1 + i % 7) * (1 + i // 7))))
            + (i % 3) for i in range(k)]


def _ids(case, n, g):
    v = case["vertices"]
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    if case["seeds"] == "flat":
        return (u * v).long().clamp_(max=v - 1).to(INDEX[case["index"]])
    place = torch.randperm(v, generator=g, device="cuda")
    return place[(u ** SKEW * v).long().clamp_(max=v - 1)].to(INDEX[case["index"]])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["dtype"]]

    def normal(shape, std=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(t)

    s = {"case": case}
    if case["op"] == "clip":
        s["grads"] = [normal((n,), 10.0 ** (-(i % 4))) for i, n in enumerate(_sizes(case))]
        # the bound that a user has set: a share of the norm that such gradients have
        power = sum(n * 10.0 ** (-2 * (i % 4)) for i, n in enumerate(_sizes(case)))
        s["max_norm"] = case["ratio"] * (math.sqrt(power) if case["norm"] == "l2" else 4.0)
    else:
        n, v, f = case["n"], case["vertices"], case["feat"]
        if case["op"] == "lookup":
            s["table"] = normal((v, f), f ** -0.5)
            s["ids"] = _ids(case, n, g)
        elif case["op"] == "lookup_grad":
            s["ids"] = _ids(case, n, g)
            s["out_grad"] = normal((n, f))
        else:
            # features of unit variance against weights that give logits of a few units
            s["feat"] = normal((n, f))
            s["weight"] = normal((v, f), 2.0 * f ** -0.5)
            labels = torch.randint(v, (n,), generator=g, device="cuda")
            skip = torch.rand(n, generator=g, device="cuda") < case["ignored"]
            s["labels"] = torch.where(skip, IGNORE, labels).to(INDEX[case["index"]])
            if case["op"] == "xent_train":
                # the mean over the batch, each sample with a weight of its own
                s["loss_grad"] = (0.5 + torch.rand(n, generator=g, device="cuda")) / n
    if own:
        s["module"] = _module(case, s)
    return s


def _module(case, s):
    """The built module that a user's program keeps."""
    from featgraph_b200 import module, te

    def like(x, name):
        return te.placeholder(tuple(x.shape), str(x.dtype).replace("torch.", ""), name)

    if case["op"] == "clip":
        m = module.GradientClipcuda()
        m.build([like(x, "Grad") for x in s["grads"]],
                {"max_norm": s["max_norm"], "norm_type": 2 if case["norm"] == "l2" else math.inf},
                {})
        return m
    if case["op"] == "lookup" or case["op"] == "lookup_grad":
        m = module.EmbeddingLookupcuda()
        m.build([te.placeholder((case["vertices"], case["feat"]), case["dtype"], "Table"),
                 like(s["ids"], "Ids")],
                {"scale": case["scale"], "with_grad": case["op"] == "lookup_grad"}, {})
        return m
    m = module.SoftmaxCrossEntropycuda()
    m.build([like(s["feat"], "Feat"), like(s["weight"], "Weight"), like(s["labels"], "Labels")],
            {"scale": case["scale"], "ignore_index": IGNORE,
             "with_grad": case["op"] == "xent_train"}, {})
    return m


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        m = state["module"]
        if op == "lookup":
            return m.run([state["table"], state["ids"]]).torch
        if op == "lookup_grad":
            return m.run_grad([state["out_grad"], state["ids"]]).torch
        if op == "clip":
            norm, clipped = m.run(state["grads"])
            return {"norm": norm.torch, "clipped": [x.torch for x in clipped]}
        feat, weight, labels = state["feat"], state["weight"], state["labels"]
        loss, lse = m.run([feat, weight, labels])
        if op == "xent":
            return {"loss": loss.torch, "lse": lse.torch}
        dfeat, dweight = m.run_grad([state["loss_grad"], feat, weight, labels, lse])
        return {"loss": loss.torch, "lse": lse.torch, "feat_grad": dfeat.torch,
                "weight_grad": dweight.torch}
    if op == "lookup":
        rows = state["table"][state["ids"].long()]
        return (rows.float() * case["scale"]).to(rows.dtype)
    if op == "lookup_grad":
        dy = state["out_grad"]
        grad = torch.zeros((case["vertices"], case["feat"]), device=dy.device)
        grad.index_add_(0, state["ids"].long(), dy.float())
        return (grad * case["scale"]).to(dy.dtype)
    if op == "clip":
        return _plain_clip(state)
    return _plain_xent(state)


def _plain_clip(state):
    case, grads = state["case"], state["grads"]
    if case["norm"] == "l2":
        norm = torch.stack([x.float().square().sum() for x in grads]).sum().sqrt()
    else:
        norm = torch.stack([x.float().abs().max() for x in grads]).max()
    share = (state["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    return {"norm": norm.reshape(1),
            "clipped": [(x.float() * share).to(x.dtype) for x in grads]}


def _plain_xent(state):
    case = state["case"]
    feat, weight, labels = state["feat"], state["weight"], state["labels"].long()
    kept = labels != IGNORE
    at = torch.where(kept, labels, 0)[:, None]
    logits = feat.float() @ weight.float().T
    logits *= case["scale"]
    top = logits.amax(1, keepdim=True)
    picked = logits.gather(1, at)
    logits -= top
    logits.exp_()
    total = logits.sum(1, keepdim=True)
    lse = top + total.log()
    loss = torch.where(kept, (lse - picked)[:, 0], 0.0)
    out = {"loss": loss, "lse": lse[:, 0]}
    if case["op"] == "xent":
        return out
    share = torch.where(kept, state["loss_grad"], 0.0)[:, None]
    dz = logits
    dz *= share / total
    dz.scatter_add_(1, at, -share)
    dz *= case["scale"]
    out["feat_grad"] = (dz @ weight.float()).to(feat.dtype)
    out["weight_grad"] = (dz.T @ feat.float()).to(weight.dtype)
    return out


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "lookup":
        return torch.index_select(s["table"].double(), 0, s["ids"].long()) * case["scale"]
    if case["op"] == "lookup_grad":
        # a one-hot matrix, transposed, times the gradient
        n, ids = case["n"], s["ids"].long()
        hot = torch.sparse_coo_tensor(torch.stack([ids, torch.arange(n, device=ids.device)]),
                                      torch.full((n,), case["scale"], dtype=torch.float64,
                                                 device=ids.device), (case["vertices"], n))
        return torch.sparse.mm(hot, s["out_grad"].double())
    if case["op"] == "clip":
        flat = torch.cat([x.double() for x in s["grads"]])
        norm = torch.linalg.vector_norm(flat, 2 if case["norm"] == "l2" else math.inf)
        coef = min(1.0, s["max_norm"] / (float(norm) + 1e-6))
        return {"norm": norm.reshape(1), "clipped": [x.double() * coef for x in s["grads"]]}
    h, w, y = s["feat"].double() * case["scale"], s["weight"].double(), s["labels"].long()
    n, v = h.shape[0], w.shape[0]
    rows = torch.arange(n, device=h.device)
    live = rows[y != IGNORE]
    step = max(1, (1 << 28) // max(n, 1))
    lse = torch.full((n,), -math.inf, dtype=torch.float64, device=h.device)
    for a in range(0, v, step):
        lse = torch.logaddexp(lse, torch.logsumexp(h @ w[a:a + step].T, 1))
    loss = torch.zeros_like(lse)
    loss[live] = lse[live] - (h[live] * w[y[live]]).sum(1)
    out = {"loss": loss, "lse": lse}
    if case["op"] == "xent":
        return out
    weight = torch.zeros_like(lse)
    weight[live] = s["loss_grad"].double()[live]
    dh, dw = torch.zeros_like(h), torch.zeros_like(w)
    for a in range(0, v, step):
        b = min(v, a + step)
        p = torch.exp(h @ w[a:b].T - lse[:, None]) * weight[:, None]
        here = live[(y[live] >= a) & (y[live] < b)]
        p[here, y[here] - a] -= weight[here]
        dh += p @ w[a:b]
        dw[a:b] = p.T @ h
    out["feat_grad"] = dh * case["scale"]
    out["weight_grad"] = dw
    return out


def _distinct(case):
    """How many of the vertices n draws reach, on average."""
    v, n = case["vertices"], case["n"]
    if case["seeds"] == "flat":
        return v * -math.expm1(n * math.log1p(-1.0 / v)) if v > 1 else 1.0
    edge = (torch.arange(v + 1, dtype=torch.float64) / v) ** (1.0 / SKEW)
    share = edge[1:] - edge[:-1]
    return float((-torch.expm1(n * torch.log1p(-share.clamp(max=1 - 1e-12)))).sum())


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "clip":
        total = sum(_sizes(case))
        return {"bytes": 2 * total * size + 4, "flops": 3 * total}
    n, v, f = case["n"], case["vertices"], case["feat"]
    index = 4 if case["index"] == "int32" else 8
    if case["op"] == "lookup":
        return {"bytes": int((_distinct(case) + n) * f * size) + n * index, "flops": n * f}
    if case["op"] == "lookup_grad":
        return {"bytes": (n + v) * f * size + n * index, "flops": n * f + v * f}
    if case["op"] == "xent":
        return {"bytes": (n + v) * f * size + n * (index + 8), "flops": 2 * n * v * f}
    # the logits' product and the two of the gradients
    return {"bytes": 2 * (n + v) * f * size + n * (index + 12), "flops": 6 * n * v * f}
