"""Measured calls of the many-class softmax cross-entropy head and of gradient clipping by the global norm.

A case is a dict of plain values.  ``op`` says which call it stands for:

  head_fwd   per-row loss and log-sum-exp of a classifier with many classes (evaluation, scoring of tokens)
  head_train the same plus the gradients of the hidden rows, the weight and the bias (one training step's head)
  norm       the global norm of a list of gradient tensors
  clip       the norm and the clipped copies of the tensors

``run`` computes a pass in its plain form, elementary torch operations in 32 bits (64 for the long sums), or -- where
``own`` is true -- through the package's kernels.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
_IGNORE = -1


def listed():
    return [
        # one token is scored: what an answer costs when every microsecond shows
        dict(name="head_fwd one row", op="head_fwd", rows=1, hidden=1024, classes=32000, dtype="bf16", bias=False, ignored=0.0),
        # a prompt is scored (perplexity): a ragged number of rows against an odd number of classes
        dict(name="head_fwd prompt", op="head_fwd", rows=777, hidden=4096, classes=50001, dtype="bf16", bias=False, ignored=0.0),
        # a few rows are trained on, all of the weight is read and its gradient written
        dict(name="head_train 16 rows", op="head_train", rows=16, hidden=4096, classes=32000, dtype="bf16", bias=False, ignored=0.0),
        # nothing divides: a padded batch (ignored rows), an odd number of classes, a bias
        dict(name="head_train ragged", op="head_train", rows=1000, hidden=1000, classes=10007, dtype="bf16", bias=True, ignored=0.2),
        # an ordinary training step at the narrow model's width
        dict(name="head_train 4096 x 65536", op="head_train", rows=4096, hidden=1024, classes=65536, dtype="bf16", bias=False, ignored=0.0),
        # the largest: the wide model's width and a large vocabulary
        dict(name="head_train 8192 x 131072", op="head_train", rows=8192, hidden=4096, classes=131072, dtype="bf16", bias=False, ignored=0.1),
        # the exact-fp32 configuration
        dict(name="head_train fp32", op="head_train", rows=1024, hidden=1024, classes=10000, dtype="fp32", bias=True, ignored=0.0),
        # the gradients of the model that this package trains: eight tensors, 13 MB, every step
        dict(name="clip model", op="clip", tensors="model", count=8, elements=0, dtype="fp32", factor=0.3),
        # norm only (logging), the widened model's 53 M gradients
        dict(name="norm wide model", op="norm", tensors="wide", count=8, elements=0, dtype="fp32", factor=0.5),
        # many small tensors of odd sizes lying in one arena, unaligned
        dict(name="clip 400 small", op="clip", tensors="arena", count=400, elements=1500000, dtype="bf16", factor=0.7),
        # fp32 and bf16 tensors together, a norm below the limit: values pass unchanged
        dict(name="clip mixed below limit", op="clip", tensors="mixed", count=40, elements=40000000, dtype="fp32", factor=2.0),
        # a large network's gradients, 0.72 G elements
        dict(name="clip large", op="clip", tensors="blocks", count=57, elements=718000000, dtype="bf16", factor=0.1),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.6:
        dtype = "fp32" if rng.random() < 0.25 else "bf16"
        most = (1 << 34) if dtype == "fp32" else (1 << 40)       # rows * hidden * classes
        while True:
            hidden = _log_uniform(rng, 64, 4096)
            if rng.random() < 0.75:
                hidden -= hidden % 8
            rows, classes = _log_uniform(rng, 1, 8192), _log_uniform(rng, 300, 131072)
            if rows * hidden * classes <= most:
                break
        return dict(op="head_fwd" if rng.random() < 0.35 else "head_train", rows=rows, hidden=hidden, classes=classes, dtype=dtype,
                    bias=rng.random() < 0.4, ignored=round(rng.uniform(0.05, 0.5), 2) if rng.random() < 0.4 else 0.0)
    tensors = "mixed" if rng.random() < 0.3 else "arena"
    return dict(op="norm" if rng.random() < 0.3 else "clip", tensors=tensors,
                count=_log_uniform(rng, 1, 60 if tensors == "mixed" else 1000), elements=_log_uniform(rng, 2000, 100000000),
                dtype="bf16" if rng.random() < 0.5 else "fp32", factor=round(math.exp(rng.uniform(math.log(0.01), math.log(3.0))), 3))


# ---------------------------------------------------------------------------------------------------------- inputs
def _head_inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, hid, v, dt = case["rows"], case["hidden"], case["classes"], _TYPES[case["dtype"]]
    w = torch.randn((v, hid), device="cuda", generator=g) * (2.0 / math.sqrt(hid))
    labels = torch.randint(0, v, (n,), device="cuda", generator=g)
    # normalised hidden rows; some of them already point at their class (a model in mid training)
    h = torch.randn((n, hid), device="cuda", generator=g)
    h += w[labels] * (3.0 * torch.rand((n, 1), device="cuda", generator=g))
    if case["ignored"]:
        drop = torch.rand((n,), device="cuda", generator=g) < case["ignored"]
        labels = torch.where(drop, torch.full_like(labels, _IGNORE), labels)
    bias = torch.randn((v,), device="cuda", generator=g) * 0.5 if case["bias"] else None
    return dict(h=h.to(dt), wT=w.to(dt), labels=labels.to(torch.int32), bias=bias, scale=1.0 / n)


def _gradients(case, seed):
    """(flat buffer or None, the list of tensors)"""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, kind = _TYPES[case["dtype"]], case["tensors"]
    if kind == "arena":     # sizes from the seedless pattern of the case: some tiny, some long, nearly all odd
        c = case["count"]
        weights = [1.0 + 9.0 * ((k * 37) % 11) ** 2 / 100.0 for k in range(c)]
        total = sum(weights)
        sizes = [max(1, int(case["elements"] * x / total) | 1) for x in weights]
        flat = torch.randn((sum(sizes),), device="cuda", generator=g)
        flat = (flat * torch.rand(flat.shape, device="cuda", generator=g) * 1e-2).to(dt)
        return flat, list(torch.split(flat, sizes))
    c1, c2, hid = (128, 256, 4096) if kind == "wide" else (32, 64, 1024)
    if kind in ("model", "wide"):
        shapes = [(49 * c2, hid), (hid, 10), (10,), (hid,), (5, 5, c1, c2), (c2,), (5, 5, 1, c1), (c1,)]
    elif kind == "mixed":
        c = case["count"]
        shapes = [(1 + 7 * (k % 5), max(1, int(case["elements"] / c / (1 + 7 * (k % 5)) * (0.5 + (k % 3) / 2)))) for k in range(c)]
    else:
        d = 2560
        shapes = [(65536, d)] + [s for _ in range(7) for s in ((d, d), (d, d), (d, d), (d, d), (4 * d, d), (d, 4 * d), (d,), (d,))]
    made = []
    for k, s in enumerate(shapes):
        t = torch.randn(s, device="cuda", generator=g) * (10.0 ** -(1 + k % 4))
        made.append(t.to(torch.bfloat16 if kind == "mixed" and k % 2 else dt))
    return None, made


def _limit(case, tensors):
    """A clipping norm that scales by about ``factor`` (or leaves the values alone where it is above one)."""
    square = sum(float(t.double().square().sum()) for t in tensors)
    return case["factor"] * math.sqrt(square)


def prepare(case, seed):
    if case["op"].startswith("head"):
        return dict(case=case, **_head_inputs(case, seed))
    flat, tensors = _gradients(case, seed)
    state = dict(case=case, flat=flat, tensors=tensors, limit=_limit(case, tensors))
    if own:     # a program keeps the plan and the clipped copies from step to step
        from distributed_tensorflow_amd.ops import GlobalNormClip
        if case["op"] == "norm":
            state["plan"] = GlobalNormClip(tensors)
        elif flat is None:
            state["plan"] = GlobalNormClip(tensors, out=[torch.empty_like(t) for t in tensors])
        else:
            state["out"] = torch.empty_like(flat)
            state["plan"] = GlobalNormClip(tensors, out=list(torch.split(state["out"], [t.numel() for t in tensors])))
    return state


# ------------------------------------------------------------------------------------------------------------ passes
def _plain_head(s):
    case = s["case"]
    n = case["rows"]
    h, w = s["h"].float(), s["wT"].float()
    z = h @ w.t()
    if s["bias"] is not None:
        z += s["bias"]
    top = z.max(dim=1, keepdim=True).values
    lse = top.squeeze(1) + torch.exp(z - top).sum(dim=1).log()
    valid = s["labels"] != _IGNORE
    safe = torch.where(valid, s["labels"], 0).long()
    rows = torch.arange(n, device=h.device)
    loss = torch.where(valid, lse - z[rows, safe], 0.0)
    if case["op"] == "head_fwd":
        return [loss, lse]
    p = torch.exp(z - lse[:, None])
    p[rows, safe] -= 1.0
    p *= torch.where(valid, s["scale"], 0.0)[:, None]
    grads = [(p @ w).to(s["h"].dtype), (p.t() @ h).to(s["wT"].dtype)]
    return [loss, lse] + grads + ([p.sum(dim=0)] if s["bias"] is not None else [])


def _own_head(s):
    from distributed_tensorflow_amd.ops import vocab_head_bwd, vocab_head_fwd
    loss, lse = vocab_head_fwd(s["h"], s["wT"], s["labels"], s["bias"], ignore_label=_IGNORE)
    if s["case"]["op"] == "head_fwd":
        return [loss, lse]
    dh, dwT, dbias = vocab_head_bwd(s["h"], s["wT"], s["labels"], lse, s["bias"], grad_scale=s["scale"], ignore_label=_IGNORE)
    return [loss, lse, dh, dwT] + ([dbias] if dbias is not None else [])


def _plain_norm(tensors):
    return torch.stack([t.float().square().sum(dtype=torch.float64) for t in tensors]).sum().sqrt()


def _plain_clip(s):
    norm = _plain_norm(s["tensors"])
    if s["case"]["op"] == "norm":
        return [norm.float()]
    factor = (s["limit"] / torch.clamp(norm, min=s["limit"])).float()
    out = [(t.float() * factor).to(t.dtype) for t in s["tensors"]]
    return [norm.float()] + (out if s["flat"] is None else [torch.cat(out)])


def _own_clip(s):
    if s["case"]["op"] == "norm":
        return [s["plan"].norm()]
    out, norm = s["plan"].clip(s["limit"])
    return [norm] + (out if s["flat"] is None else [s["out"]])


def run(state):
    if state["case"]["op"].startswith("head"):
        return _own_head(state) if own else _plain_head(state)
    return _own_clip(state) if own else _plain_clip(state)


# ------------------------------------------------------------------------------------------------------ floor, truth
def _sizes(case):
    """bytes of the tensors of a clipping case"""
    flat, tensors = 0, case["tensors"]
    if tensors == "arena":
        c = case["count"]
        weights = [1.0 + 9.0 * ((k * 37) % 11) ** 2 / 100.0 for k in range(c)]
        flat = sum(max(1, int(case["elements"] * x / sum(weights)) | 1) for x in weights)
    elif tensors == "mixed":
        c = case["count"]
        sizes = [(1 + 7 * (k % 5)) * max(1, int(case["elements"] / c / (1 + 7 * (k % 5)) * (0.5 + (k % 3) / 2))) for k in range(c)]
        return sum(n * (2 if k % 2 or case["dtype"] == "bf16" else 4) for k, n in enumerate(sizes)), sum(sizes)
    elif tensors == "blocks":
        flat = 65536 * 2560 + 7 * (12 * 2560 * 2560 + 2 * 2560)
    else:
        c1, c2, hid = (128, 256, 4096) if tensors == "wide" else (32, 64, 1024)
        flat = 49 * c2 * hid + 11 * hid + 10 + 25 * c1 * c2 + c2 + 26 * c1
    return flat * (2 if case["dtype"] == "bf16" else 4), flat


def work(case):
    if case["op"].startswith("head"):
        n, hid, v, e = case["rows"], case["hidden"], case["classes"], 2 if case["dtype"] == "bf16" else 4
        once = (n + v) * hid * e + 4 * n + (4 * v if case["bias"] else 0)
        if case["op"] == "head_fwd":
            return {"bytes": once + 8 * n, "flops": 2.0 * n * hid * v}
        return {"bytes": 2 * once + 4 * n, "flops": 6.0 * n * hid * v}
    size, n = _sizes(case)
    return {"bytes": size, "flops": 2.0 * n} if case["op"] == "norm" else {"bytes": 2 * size, "flops": 3.0 * n}


def _exact_head(case, seed):
    s = _head_inputs(case, seed)
    n, v, hid = case["rows"], case["classes"], case["hidden"]
    h, labels = s["h"].double(), s["labels"].long()
    step = max(1, min(v, (1 << 28) // n))
    cuts = [(a, min(v, a + step)) for a in range(0, v, step)]

    def scores(a, b):
        z = torch.matmul(h, s["wT"][a:b].double().transpose(0, 1))
        return z if s["bias"] is None else z + s["bias"][a:b].double()

    lse = torch.logsumexp(torch.stack([torch.logsumexp(scores(a, b), 1) for a, b in cuts], 1), 1)
    keep = labels.ne(_IGNORE)
    at = labels.clamp(min=0)
    picked = (h * s["wT"].double()[at]).sum(1) + (0.0 if s["bias"] is None else s["bias"].double()[at])
    loss = (lse - picked) * keep
    if case["op"] == "head_fwd":
        return [loss, lse]
    weight = keep.double() * s["scale"]
    dh, dw = torch.zeros((n, hid), dtype=torch.float64, device="cuda"), torch.empty((v, hid), dtype=torch.float64, device="cuda")
    db = torch.empty((v,), dtype=torch.float64, device="cuda")
    for a, b in cuts:
        d = (scores(a, b) - lse.unsqueeze(1)).exp()
        mine = torch.nonzero((at >= a) & (at < b)).squeeze(1)
        d.index_put_((mine, at[mine] - a), torch.full((mine.numel(),), -1.0, dtype=torch.float64, device="cuda"), accumulate=True)
        d = d * weight.unsqueeze(1)
        dh.addmm_(d, s["wT"][a:b].double())
        dw[a:b] = torch.matmul(d.transpose(0, 1), h)
        db[a:b] = d.sum(0)
    return [loss, lse, dh, dw] + ([] if s["bias"] is None else [db])


def exact(case, seed):
    if case["op"].startswith("head"):
        return _exact_head(case, seed)
    flat, tensors = _gradients(case, seed)
    norm = math.sqrt(math.fsum(float(torch.linalg.vector_norm(t.reshape(-1).double()).square()) for t in tensors))
    if case["op"] == "norm":
        return [torch.tensor(norm, dtype=torch.float64)]
    limit = _limit(case, tensors)
    by = limit / norm if norm > limit else 1.0
    clipped = [flat.double() * by] if flat is not None else [t.double() * by for t in tensors]
    return [torch.tensor(norm, dtype=torch.float64)] + clipped
