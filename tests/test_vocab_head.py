"""The many-class softmax cross-entropy head (ops/vocab_head.py, csrc/kernels/vocab_head.hip) against the formula in 64 bits.

Bounds (u = 2^-24, half = half a rounding step of the operand type):
  logits    a sum of H products, the rounding errors of its partial sums (each at most u times S_iv = sum_k |h_ik w_vk|) wander:
            e_z = 8 sqrt(H + 64) u S; the largest over a row counts for the row's log-sum-exp (fp32 products are themselves
            off by 2^-21 = 8 u at most, which the 64 covers)
  lse       e_lse = max_v e_z + 8 u (1 + |lse|)              loss  e_lse + e_z + 8 u (1 + |lse| + |z_y|)
  d         |s| (p (e_z + e_lse + 8 u (1 + |z| + |lse|)) + 2 u), and the rounding to the operand type: half |d|
  products  every error of d times the other factor, summed, plus the accumulation 8 sqrt(terms) u sum |d| |w|, plus half of
            the result for its own rounding
The sum of d's own rounding errors is bounded by their absolute sum (no cancellation assumed)."""
import math

import pytest
import torch

from distributed_tensorflow_amd.ops import vocab_head_bwd, vocab_head_fwd

DEV = "cuda"
gpu = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def make(n, hidden, classes, dtype="bf16", bias=False, ignored=0.0, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    w = torch.randn((classes, hidden), device=DEV, generator=g) * (2.0 / math.sqrt(hidden))
    labels = torch.randint(0, classes, (n,), device=DEV, generator=g)
    h = torch.randn((n, hidden), device=DEV, generator=g) + w[labels] * torch.rand((n, 1), device=DEV, generator=g) * 2
    if ignored:
        labels = torch.where(torch.rand((n,), device=DEV, generator=g) < ignored, torch.full_like(labels, -1), labels)
    b = torch.randn((classes,), device=DEV, generator=g) * 0.5 if bias else None
    return h.to(TYPES[dtype]), w.to(TYPES[dtype]), labels.to(torch.int32), b


class Exact:
    """The formula in fp64 and the bounds above."""

    def __init__(self, h, w, labels, bias=None, grad_scale=1.0, row_scale=None, ignore=-1):
        self.h, self.w = h.double(), w.double()
        n, hidden = h.shape
        lab = labels.long()
        self.live = lab != ignore
        y = lab.clamp(0, w.shape[0] - 1)
        z = self.h @ self.w.t()
        if bias is not None:
            z = z + bias.double()
        ez = 8 * math.sqrt(hidden + 64) * U * (self.h.abs() @ self.w.abs().t())
        if bias is not None:
            ez = ez + 2 * U * torch.nan_to_num(bias.double().abs(), posinf=0.0)
        self.lse = torch.logsumexp(z, 1)
        zy = z.gather(1, y[:, None]).squeeze(1)
        self.e_lse = ez.max(1).values + 8 * U * (1 + self.lse.abs())
        self.loss = torch.where(self.live, self.lse - zy, 0.0)
        self.e_loss = self.e_lse + ez.gather(1, y[:, None]).squeeze(1) + 8 * U * (1 + self.lse.abs() + zy.abs())
        s = torch.full((n,), float(grad_scale), dtype=torch.float64, device=h.device)
        if row_scale is not None:
            s = s * row_scale.double()
        s = torch.where(self.live, s, 0.0)[:, None]
        p = torch.exp(z - self.lse[:, None])
        d = p.clone()
        d[torch.arange(n, device=h.device), y] -= 1.0
        self.d = s * d
        zf = torch.nan_to_num(z, neginf=0.0)
        self.e_d = s.abs() * (p * (ez + self.e_lse[:, None] + 8 * U * (1 + zf.abs() + self.lse.abs()[:, None])) + 2 * U)
        self.half = half_step(h.dtype)

    def _product(self, d, e_d, x, dtype):
        got = d @ x
        e = (e_d + (self.half if self.half > U else 0.0) * d.abs() + 8 * math.sqrt(d.shape[1]) * U * d.abs()) @ x.abs()
        return got, e + half_step(dtype) * (got.abs() + e)

    def dh(self):
        return self._product(self.d, self.e_d, self.w, TYPES["bf16"] if self.half > U else TYPES["fp32"])

    def dw(self, dtype):
        return self._product(self.d.t(), self.e_d.t(), self.h, dtype)

    def db(self):
        return self.d.sum(0), self.e_d.sum(0) + 8 * math.sqrt(self.d.shape[0]) * U * self.d.abs().sum(0) + U * self.d.sum(0).abs()


def within(got, want, bound, what):
    over = (got.double() - want).abs() - bound
    assert bool((over <= 0).all()), f"{what}: {float(over.max()):.3g} beyond its bound (largest bound {float(bound.max()):.3g})"


def check_all(h, w, labels, bias, grad_scale=1.0, row_scale=None, dw_dtype=None, piece=0, ignore=-1):
    x = Exact(h, w, labels, bias, grad_scale, row_scale, ignore)
    loss, lse = vocab_head_fwd(h, w, labels, bias, ignore_label=ignore)
    within(lse, x.lse, x.e_lse, "lse")
    within(loss, x.loss, x.e_loss, "loss")
    dwT = torch.full(w.shape, 9.0, dtype=dw_dtype, device=DEV) if dw_dtype else None
    dh, dw, db = vocab_head_bwd(h, w, labels, lse, bias, grad_scale=grad_scale, row_scale=row_scale, ignore_label=ignore, dwT=dwT,
                                piece=piece)
    assert dh.dtype == h.dtype and dw.dtype == (dw_dtype or w.dtype) and dh.shape == h.shape and dw.shape == w.shape
    within(dh, *x.dh(), "dh")
    within(dw, *x.dw(dw.dtype), "dw")
    if bias is None:
        assert db is None
    else:
        within(db, *x.db(), "db")
    return loss, lse, dh, dw, db


# ---------------------------------------------------------------------------------------------------- refusals (no GPU)
def test_refuses_what_it_does_not_take():
    h, w, y = torch.zeros(4, 8), torch.zeros(16, 8), torch.zeros(4, dtype=torch.int32)
    bad = [
        (TypeError, "both be bf16", (h.half(), w.half(), y), {}),
        (TypeError, "both be bf16", (h.bfloat16(), w, y), {}),
        (ValueError, "hidden units", (h, torch.zeros(16, 9), y), {}),
        (ValueError, "contiguous rows", (h, torch.zeros(8, 16).t(), y), {}),
        (ValueError, "contiguous rows", (torch.zeros(4, 2, 8), w, y), {}),
        (ValueError, "share memory", (torch.zeros(1, 8).expand(4, 8), w, y), {}),
        (ValueError, "labels", (h, w, y.long()), {}),
        (ValueError, "labels", (h, w, y[:3]), {}),
        (ValueError, "bias", (h, w, y, torch.zeros(15)), {}),
        (ValueError, "bias", (h, w, y, torch.zeros(16).bfloat16()), {}),
        (ValueError, "classes expected", (h, torch.zeros(0, 8), y), {}),
        (ValueError, "classes expected", (torch.zeros(4, 0), torch.zeros(16, 0), y), {}),
        (ValueError, "ignore_label", (h, w, y), dict(ignore_label=1 << 31)),
        (ValueError, "may be at most", (torch.zeros(2, (1 << 20) + 1), torch.zeros(2, (1 << 20) + 1), y[:2]), {}),
        (ValueError, "at most", (torch.zeros((1 << 20) + 1, 1), torch.zeros(2, 1), torch.zeros((1 << 20) + 1, dtype=torch.int32)), {}),
        (ValueError, "GPU tensors expected", (h, w, y), {}),
    ]
    for kind, text, args, kw in bad:
        with pytest.raises(kind, match=text):
            vocab_head_fwd(*args, **kw)


@gpu
def test_backward_refusals(gpu_lib):
    h, w, y, b = make(4, 8, 16, "fp32", bias=True)
    lse = torch.zeros(4, device=DEV)
    bad = [
        ("lse is missing", dict(lse=None)),
        ("lse must be", dict(lse=lse.bfloat16())),
        ("row_scale", dict(row_scale=torch.ones(5, device=DEV))),
        ("piece", dict(piece=-1)),
        ("dh must be", dict(dh=torch.zeros(4, 9, device=DEV))),
        ("dh must be", dict(dh=torch.zeros(4, 8, device=DEV).bfloat16())),
        ("dwT must be", dict(dwT=torch.zeros(16 * 8 + 1, device=DEV)[1:].view(16, 8))),
        ("dbias must be", dict(dbias=torch.zeros(16, device=DEV).double())),
        ("shares memory", dict(dh=h)),
        ("shares memory", dict(dwT=w)),
    ]
    for text, kw in bad:
        args = {**dict(lse=lse), **kw}
        with pytest.raises(ValueError, match=text):
            vocab_head_bwd(h, w, y, args.pop("lse"), b, **args)
    with pytest.raises(ValueError, match="dbias without"):
        vocab_head_bwd(h, w, y, lse, dbias=torch.zeros(16, device=DEV))
    with pytest.raises(ValueError, match="labels is on cpu"):
        vocab_head_fwd(h, w, y.cpu())


@gpu
def test_native_entries_refuse(gpu_lib):
    h, w, y, _ = make(4, 8, 16, "fp32")
    out = torch.zeros(64, device=DEV)
    ws = torch.zeros(1 << 20, dtype=torch.uint8, device=DEV)
    s = torch.cuda.current_stream().cuda_stream
    p = lambda t: t.data_ptr()  # noqa: E731
    need = gpu_lib.dtf_vocab_head_workspace(0, 0, p(h), 8, p(w), 8, 4, 8, 16, 0, 0)
    assert 0 < need <= ws.numel()

    def fwd(**kw):
        a = {**dict(dt=0, h=p(h), ldh=8, w=p(w), ldw=8, n=4, H=8, V=16, ws=p(ws), nb=need, loss=p(out)), **kw}
        return gpu_lib.dtf_vocab_head_fwd(a["dt"], a["h"], a["ldh"], a["w"], a["ldw"], None, p(y), a["n"], a["H"], a["V"], -1,
                                          a["loss"], p(out), a["ws"], a["nb"], s)

    assert fwd(nb=need - 1) == -2
    for bad in (dict(dt=2), dict(h=None), dict(w=None), dict(ldh=7), dict(ldw=7), dict(n=0), dict(n=(1 << 20) + 1), dict(H=0), dict(V=0),
                dict(ws=None), dict(ws=p(ws) + 16), dict(loss=None), dict(h=p(h) + 2)):
        assert fwd(**bad) == -3, bad


# ----------------------------------------------------------------------------------------------------------- values
SHAPES = [(1, 64, 300), (2, 8, 1), (3, 16, 2), (1, 1000, 257), (37, 72, 1000), (128, 256, 513), (257, 1000, 777), (300, 33, 511),
          (513, 128, 2049), (16, 2048, 600), (64, 1, 64), (130, 40, 255), (15, 136, 4099), (700, 24, 31)]


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n,hidden,classes", SHAPES)
def test_against_the_formula(gpu_lib, n, hidden, classes, dtype):
    check_all(*make(n, hidden, classes, dtype, seed=n + classes), grad_scale=1.0 / n)


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n,hidden,classes,piece", [(37, 72, 1000, 256), (257, 64, 777, 512), (300, 33, 1500, 300), (5, 2048, 600, 256)])
def test_pieces_bias_ignored_rows_and_row_scales(gpu_lib, n, hidden, classes, piece, dtype):
    h, w, y, b = make(n, hidden, classes, dtype, bias=True, ignored=0.3, seed=11)
    scale = torch.rand(n, device=DEV) + 0.1
    scale[0] = 0.0
    one = check_all(h, w, y, b, grad_scale=0.25, row_scale=scale, piece=piece)
    whole = check_all(h, w, y, b, grad_scale=0.25, row_scale=scale)
    assert torch.equal(one[3], whole[3]) and torch.equal(one[4], whole[4])       # dw and db do not depend on the pieces
    again = check_all(h, w, y, b, grad_scale=0.25, row_scale=scale, piece=piece)
    assert all(torch.equal(a, c) for a, c in zip(one, again))                    # and nothing on the run
    assert bool((one[2][y == -1] == 0).all())
    check_all(h, w, y, b, dw_dtype=torch.float32, piece=piece)


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n,hidden,classes,piece", [
    (300, 64, 32000, 0),        # 256 x 128 tiles
    (1000, 40, 10007, 0),       # 192 x 256
    (777, 64, 50001, 0),        # three rounds of 256 x 256, the other classes in small tiles
    (2049, 72, 20011, 8192),    # pieces tiled differently
    (130, 8, 70001, 0),
    (5, 48, 30000, 0),          # from here on what few rows and classes run: 64 x 32 tiles (fp32)
    (2, 40, 60001, 0), (40, 24, 60001, 0), (100, 64, 20011, 0),     # 64 x 64
    (150, 72, 20011, 0), (200, 72, 20011, 0)])                      # 128 x 64
def test_every_tiling_of_the_logits(gpu_lib, n, hidden, classes, piece, dtype):
    h, w, y, b = make(n, hidden, classes, dtype, bias=True, ignored=0.1, seed=classes)
    y[:4] = torch.tensor([classes - 1, classes - 2, 0, 255], dtype=torch.int32, device=DEV)[:n]
    check_all(h, w, y, b, grad_scale=1.0 / n, piece=piece)


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n,hidden,classes", [
    (1100, 1800, 8000),         # dh and dw in 256 x 256 tiles
    (1100, 1800, 18011),        # dw in 128 x 128 tiles
    (300, 600, 40003),          # dh in 128 x 128 tiles and slabs
    (700, 1000, 20011),         # both in 128 x 128 tiles
    (1030, 2050, 4100)])        # a few rows, hidden units and classes over
def test_every_tiling_of_the_gradients(gpu_lib, n, hidden, classes, dtype):
    h, w, y, b = make(n, hidden, classes, dtype, bias=True, ignored=0.1, seed=hidden)
    check_all(h, w, y, b, grad_scale=1.0 / n)


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n,hidden,classes", [(1, 6, 40), (3, 74, 500), (70, 1002, 777), (300, 38, 3001), (520, 202, 2049), (150, 1001, 300)])
def test_rows_that_start_on_four_bytes(gpu_lib, n, hidden, classes, dtype):
    """Weights whose rows are no multiple of 16 bytes, read where they lie: at the end of their memory NaN follow."""
    h, w, y, b = make(n, hidden, classes, dtype, bias=True, ignored=0.1 if n > 1 else 0.0, seed=hidden)
    base = check_all(h, w, y, b, grad_scale=1.0 / n)
    room = torch.full((classes * hidden + 64,), math.nan, device=DEV).to(w.dtype)
    for start in (0, 2, 6):
        v = room[start:start + classes * hidden].view(classes, hidden)
        v.copy_(w)
        loss, lse = vocab_head_fwd(h, v, y, b)
        again = (loss, lse) + vocab_head_bwd(h, v, y, lse, b, grad_scale=1.0 / n)
        assert all(torch.equal(a, c) for a, c in zip(base, again)), start
        v.fill_(math.nan)


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_strided_and_unaligned_rows(gpu_lib, dtype):
    h, w, y, b = make(70, 96, 400, dtype, bias=True, seed=4)
    base = check_all(h, w, y, b)
    for off, pad in ((8, 24), (3, 7), (0, 1)):
        big_h = torch.full((70, 96 + off + pad), math.nan, device=DEV).to(h.dtype)
        big_w = torch.full((400, 96 + off + pad), math.nan, device=DEV).to(h.dtype)
        big_h[:, off:off + 96], big_w[:, off:off + 96] = h, w
        hv, wv = big_h[:, off:off + 96], big_w[:, off:off + 96]
        loss, lse = vocab_head_fwd(hv, wv, y, b)
        grads = vocab_head_bwd(hv, wv, y, lse, b)
        assert all(torch.equal(a, c) for a, c in zip(base, (loss, lse) + grads)), (off, pad)


@gpu
def test_outputs_in_an_arena(gpu_lib):
    """Gradients written into views of one buffer, nothing around them touched."""
    h, w, y, b = make(33, 40, 101, "bf16", bias=True, seed=5)
    base = check_all(h, w, y, b, dw_dtype=torch.float32)
    flat = torch.full((16 + 101 * 40 + 16 + 104 + 16,), 7.0, device=DEV)
    dw, db = flat[16:16 + 4040].view(101, 40), flat[16 + 4040 + 16:16 + 4040 + 16 + 101]
    buf = torch.full((33 * 40 + 32,), 7.0, device=DEV).bfloat16()
    dh = buf[16:16 + 33 * 40].view(33, 40)
    _, lse = vocab_head_fwd(h, w, y, b)
    vocab_head_bwd(h, w, y, lse, b, dh=dh, dwT=dw, dbias=db)
    assert torch.equal(dh, base[2]) and torch.equal(dw, base[3]) and torch.equal(db, base[4])
    assert bool((flat[:16] == 7).all()) and bool((flat[16 + 4040:16 + 4040 + 16] == 7).all()) and bool((flat[16 + 4040 + 16 + 101:] == 7).all())
    assert bool((buf[:16] == 7).all()) and bool((buf[16 + 33 * 40:] == 7).all())
    only_h = vocab_head_bwd(h, w, y, lse, b, need_dwT=False)
    assert only_h[1] is None and torch.equal(only_h[0], base[2])
    only_w = vocab_head_bwd(h, w, y, lse, need_dh=False)
    assert only_w[0] is None and only_w[2] is None


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_masked_classes_infinities_and_padding(gpu_lib, dtype):
    h, w, y, b = make(50, 64, 700, dtype, bias=True, seed=6)
    # classes from 500 on do not exist (a padded vocabulary): whole tiles of -inf
    b[500:] = -math.inf
    b[0] = torch.finfo(torch.float32).min
    y = torch.where(y >= 500, y - 400, y)
    y = torch.where(y == 0, torch.ones_like(y), y)
    _, lse, dh, dw, db = check_all(h, w, y, b)
    assert bool((dw[500:] == 0).all()) and bool((db[500:] == 0).all()) and bool((db[0] == 0).all())
    # padding rows may hold anything
    z = h.clone()
    y2 = y.clone()
    y2[7], y2[9], y2[49] = -1, -1, -1
    z[7], z[9], z[49] = math.nan, math.inf, 3e38
    good = h.clone()
    good[7], good[9], good[49] = 0, 0, 0
    loss, lse2 = vocab_head_fwd(z, w, y2, b)
    got = vocab_head_bwd(z, w, y2, lse2, b)
    loss_g, lse_g = vocab_head_fwd(good, w, y2, b)
    want = vocab_head_bwd(good, w, y2, lse_g, b)
    assert torch.equal(loss, loss_g) and all(torch.equal(a, c) for a, c in zip(got, want))
    # another ignored value; every row ignored
    check_all(h, w, torch.where(y2 < 0, torch.full_like(y2, 555), y2), b, ignore=555)
    none = torch.full_like(y, -1)
    loss, lse3 = vocab_head_fwd(h, w, none, b)
    assert bool((loss == 0).all()) and all(bool((t == 0).all()) for t in vocab_head_bwd(h, w, none, lse3, b))


@gpu
def test_a_label_outside_the_classes_is_loud(gpu_lib):
    h, w, y, _ = make(20, 32, 300, "fp32", seed=7)
    for bad in (300, 1 << 30, -2, -(1 << 31)):
        y2 = y.clone()
        y2[3] = bad
        loss, lse = vocab_head_fwd(h, w, y2)
        dh, dw, _ = vocab_head_bwd(h, w, y2, lse)
        assert bool(torch.isnan(loss[3])) and int(torch.isnan(loss).sum()) == 1
        assert bool(torch.isnan(dh[3]).all()) and not bool(torch.isnan(dh[:3]).any()) and not bool(torch.isnan(dh[4:]).any())
        assert bool(torch.isnan(dw).all())


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_nan_and_infinite_logits(gpu_lib, dtype):
    h, w, y, _ = make(6, 32, 600, dtype, seed=8)
    h[1, 3] = math.nan
    loss, _ = vocab_head_fwd(h, w, y)
    assert bool(torch.isnan(loss[1])) and int(torch.isnan(loss).sum()) == 1
    # one class alone has a label, the others are -inf: loss 0, gradient 0
    b = torch.full((600,), -math.inf, device=DEV)
    b[5] = 0.0
    h, w, _, _ = make(6, 32, 600, dtype, seed=9)
    five = torch.full((6,), 5, dtype=torch.int32, device=DEV)
    loss, lse = vocab_head_fwd(h, w, five, b)
    assert float(loss.abs().max()) <= 8 * U * (1 + float(lse.abs().max()))
    # the label itself is masked: the loss is infinite, the gradient still finite
    loss, lse = vocab_head_fwd(h, w, torch.full_like(five, 6), b)
    assert bool(torch.isinf(loss).all())
    assert all(bool(torch.isfinite(t).all()) for t in vocab_head_bwd(h, w, torch.full_like(five, 6), lse, b))


@gpu
def test_large_logits(gpu_lib):
    """Logits of +-1e4: nothing overflows, and the bounds (relative to the sums of products) hold."""
    h, w, y, b = make(40, 64, 900, "fp32", bias=True, seed=10)
    check_all(h * 3000.0, w, y, b)
    check_all(h * 1e-20, w, y, b)


@gpu
def test_no_rows(gpu_lib):
    h, w, _, b = make(1, 16, 50, "bf16", bias=True)
    y = torch.zeros(0, dtype=torch.int32, device=DEV)
    loss, lse = vocab_head_fwd(h[:0], w, y, b)
    dh, dw, db = vocab_head_bwd(h[:0], w, y, lse, b)
    assert loss.shape == (0,) and dh.shape == (0, 16) and bool((dw == 0).all()) and bool((db == 0).all())


@gpu
def test_gradients_against_differences(gpu_lib):
    """Central differences of the summed loss along random directions.  Step e = 2^-6 on directions that move no logit by
    more than 1: the third derivative along them is at most n (a cumulant of a variable within [-1, 1] is at most 2), so the
    difference is off by at most e^2 n / 3; the losses are off by their rounding, at most n (e_loss) / e."""
    n, hidden, classes = 8, 16, 300
    h, w, y, b = make(n, hidden, classes, "fp32", bias=True, seed=12)
    x = Exact(h, w, y, b)
    _, lse = vocab_head_fwd(h, w, y, b)
    dh, dw, db = vocab_head_bwd(h, w, y, lse, b)
    e = 2.0 ** -6
    g = torch.Generator(device=DEV).manual_seed(1)
    for k, (t, grad) in enumerate(((h, dh), (w, dw), (b, db))):
        v = torch.randn(t.shape, device=DEV, generator=g)
        moved = (v @ w.t()) if k == 0 else (h @ v.t()) if k == 1 else v
        v = v / moved.abs().max()

        def loss(sign):
            args = [h, w, y, b]
            args[(0, 1, 3)[k]] = t + sign * e * v
            return vocab_head_fwd(*args)[0].double().sum()

        diff = float(loss(1) - loss(-1)) / (2 * e)
        want = float((grad.double() * v.double()).sum())
        assert abs(diff - want) <= e * e * n / 3 + float(x.e_loss.sum()) / e


@gpu
def test_offsets_beyond_32_bits(gpu_lib):
    """A weight of 4.9 GB: classes at its end are read, and their gradient written, where they lie."""
    n, hidden, classes = 4, 4096, 600_000
    w = torch.zeros((classes, hidden), dtype=torch.bfloat16, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(3)
    h = torch.randn((n, hidden), device=DEV, generator=g).bfloat16()
    places = torch.tensor([0, 1, 300_001, 524_288, 599_998, 599_999], device=DEV)
    w[places] = (torch.randn((6, hidden), device=DEV, generator=g) * 0.05).bfloat16()
    y = torch.tensor([599_999, 524_288, 1, 17], dtype=torch.int32, device=DEV)
    loss, lse = vocab_head_fwd(h, w, y)
    z = h.double() @ w[places].double().t()
    want = torch.log(torch.exp(z).sum(1) + (classes - 6))
    assert float((lse.double() - want).abs().max()) <= 1e-4       # the bound of Exact at these sums: 8 sqrt(4160) u 130 = 4e-3
    _, dw, _ = vocab_head_bwd(h, w, y, lse, need_dh=True)
    p = torch.exp(z - want[:, None])
    for k, c in enumerate(places.tolist()):
        d = p[:, k] - (y == c).double()
        ref = d @ h.double()
        assert float((dw[c].double() - ref).abs().max()) <= (2.0 ** -7) * float((d.abs() @ h.double().abs()).max())
    assert float((dw[17].double() - (torch.exp(-want) - (y == 17).double()) @ h.double()).abs().max()) <= 2.0 ** -7 * float(h.abs().max())
    del w, dw
    torch.cuda.empty_cache()


@gpu
def test_offsets_beyond_32_bits_many_rows(gpu_lib):
    """The same for rows enough to run the large tiles: all classes but the last two have a weight of zero, so every row's
    log-sum-exp is log(classes - 2 + exp(z_a) + exp(z_b)); the gradient's rows of those two, and of one in the middle."""
    n, hidden, classes = 200, 4096, 600_000
    g = torch.Generator(device=DEV).manual_seed(5)
    w = torch.zeros((classes, hidden), dtype=torch.bfloat16, device=DEV)
    w[-2:] = (torch.randn((2, hidden), device=DEV, generator=g) * 0.05).bfloat16()
    h = torch.randn((n, hidden), device=DEV, generator=g).bfloat16()
    y = torch.where(torch.arange(n, device=DEV) % 2 == 0, classes - 1, 300_001).to(torch.int32)
    loss, lse = vocab_head_fwd(h, w, y)
    hd = h.double()
    z = hd @ w[-2:].double().t()
    want = torch.log(torch.exp(z).sum(1) + (classes - 2))
    e_z = 8 * math.sqrt(hidden + 64) * U * (hd.abs() @ w[-2:].double().abs().t())
    e_lse = e_z.max(1).values + 8 * U * (1 + want)
    within(lse, want, e_lse, "lse")
    within(loss, torch.where(y == classes - 1, want - z[:, 1], want), 2 * e_lse + 8 * U * z.abs().sum(1), "loss")
    dh, dw, _ = vocab_head_bwd(h, w, y, lse)
    half = half_step(torch.bfloat16)
    cols = torch.stack([torch.exp(-want), torch.exp(z[:, 0] - want), torch.exp(z[:, 1] - want)], 1)
    hit = torch.stack([y == 300_001, y == classes - 2, y == classes - 1], 1).double()
    d = cols - hit
    e_d = cols * (2 * e_lse + 8 * U * (1 + want))[:, None] + 2 * U + half * d.abs()
    got = d.t() @ hd
    e = (e_d + 8 * math.sqrt(n) * U * d.abs()).t() @ hd.abs()
    within(dw[[300_001, classes - 2, classes - 1]], got, e + half * (got.abs() + e), "dw")
    # dh: only the last two classes' weights are not zero
    d, e_d = d[:, 1:], e_d[:, 1:] + 8 * math.sqrt(classes) * U * d[:, 1:].abs()
    got, e = d @ w[-2:].double(), e_d @ w[-2:].double().abs()
    within(dh, got, e + half * (got.abs() + e), "dh")
    del w, dw
    torch.cuda.empty_cache()


@gpu
def test_stride_of_a_single_row_says_nothing(gpu_lib):
    big = torch.zeros((2, (1 << 20) + 64), device=DEV)
    h, w, y, _ = make(1, 32, 90, "fp32", seed=2)
    big[0, :32] = h[0]
    view = big[:1, :32]
    assert view.stride(0) > 1 << 20
    assert torch.equal(vocab_head_fwd(view, w, y)[1], vocab_head_fwd(h, w, y)[1])
    assert torch.equal(vocab_head_fwd(h, view, torch.zeros_like(y))[1], vocab_head_fwd(h, h, torch.zeros_like(y))[1])


def without_own_rounding(x, grad_scale, kept):
    """(dw, bound) in fp32 where d, relative to grad_scale, is rounded to bf16 once -- by its distance to the nearest bf16 value,
    which changes by no more than d itself does -- or (kept) carries its rounding error in a second bf16 value: half^2."""
    d1, e1 = x.d / grad_scale, x.e_d / grad_scale
    far = x.half * x.half * d1.abs() if kept else (d1.float().bfloat16().double() - d1).abs() + U * d1.abs()
    d, e_d = x.d.t(), (grad_scale * (2 * e1 + far)).t()
    got = d @ x.h
    e = (e_d + 8 * math.sqrt(2 * d.shape[1]) * U * d.abs()) @ x.h.abs()
    return got, e + U * (got.abs() + e)


@gpu
@pytest.mark.parametrize("n", [300, 1000])
def test_the_common_factor_is_not_rounded_into_the_gradient(gpu_lib, n):
    """Classes that are all alike: a label's d is -(1 - 1/classes), next to a bf16 value, and would be off by 0.39 % in every row
    if it were rounded after its product with a factor that lies halfway between two bf16 values."""
    s = (1 + 2.0 ** -8) / 1024
    h, w, y, b = make(n, 64, 3000, "bf16", seed=n)
    h = h * 0.01
    x = Exact(h, w, y, b, grad_scale=s)
    _, lse = vocab_head_fwd(h, w, y, b)
    dw = torch.empty(w.shape, device=DEV)
    vocab_head_bwd(h, w, y, lse, b, grad_scale=s, dwT=dw)
    got, e = without_own_rounding(x, s, False)
    within(dw, got, e, "dw")
    assert float(e[y.long()].abs().median()) < 2e-3 * float(got[y.long()].abs().median())


@gpu
@pytest.mark.parametrize("n,classes,piece", [(1, 400, 0), (1, 2000, 256), (5, 1111, 0), (17, 300, 0), (32, 4099, 1024)])
def test_few_rows_keep_what_rounding_drops(gpu_lib, n, classes, piece):
    h, w, y, b = make(n, 96, classes, "bf16", bias=True, ignored=0.1 if n > 1 else 0.0, seed=n + classes)
    s = 0.3
    x = Exact(h, w, y, b, grad_scale=s)
    _, lse = vocab_head_fwd(h, w, y, b)
    dw = torch.empty(w.shape, device=DEV)
    dh, _, _ = vocab_head_bwd(h, w, y, lse, b, grad_scale=s, dwT=dw, piece=piece)
    got, e = without_own_rounding(x, s, True)
    within(dw, got, e, "dw")
    got = x.d @ x.w
    e = (2 * x.e_d + (x.half ** 2 + 8 * math.sqrt(2 * classes) * U) * x.d.abs()) @ x.w.abs()
    within(dh, got, e + x.half * (got.abs() + e), "dh")


# ---------------------------------------------------------------------------------------------- streams and graphs
@gpu
@pytest.mark.parametrize("n,hidden,classes,dtype", [(130, 64, 900, "bf16"), (5, 64, 900, "bf16"), (20, 37, 700, "fp32"),
                                                    (40, 33, 900, "bf16"), (300, 72, 2100, "fp32")])
def test_graph_replays_and_streams(gpu_lib, n, hidden, classes, dtype):
    a = make(n, hidden, classes, dtype, bias=True, ignored=0.2, seed=20)
    graphs, results = [], []
    for _ in range(2):
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            loss, lse = vocab_head_fwd(*a)
            results.append((loss, lse) + vocab_head_bwd(a[0], a[1], a[2], lse, a[3], piece=256))
        graphs.append(g)
    for rep in range(3):
        fresh = make(n, hidden, classes, dtype, bias=True, ignored=0.2, seed=30 + rep)
        for t, f in zip(a, fresh):
            t.copy_(f)
        loss, lse = vocab_head_fwd(*a)
        want = (loss, lse) + vocab_head_bwd(a[0], a[1], a[2], lse, a[3], piece=256)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for r in results:
            assert all(torch.equal(x, y) for x, y in zip(r, want))
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            loss, lse = vocab_head_fwd(*a)
            got.append((loss, lse) + vocab_head_bwd(a[0], a[1], a[2], lse, a[3], piece=256))
    torch.cuda.synchronize()
    for r in got:
        assert all(torch.equal(x, y) for x, y in zip(r, want))
