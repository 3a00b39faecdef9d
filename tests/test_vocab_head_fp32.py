"""The fp32 products of the many-class head, one product at a time (csrc/kernels/vocab_head.hip: three bf16 parts of each value).

The sums of test_vocab_head.py are bounded by the errors of whole softmax gradients, next to which a part that is missing does not
show.  Here d is known exactly: with a log-sum-exp of 1000 every exponential is zero, so d is -row_scale at the label and zero
elsewhere.  Then every element of dh is ONE product, row_scale_i * w[y_i][k], and dw sums one product for each row of a class.

Bound, u = 2^-24: 8 u of a product for the parts that are left out (2^-21), and of the running sum 2 u for each of the six
instructions that add to it (rounding or truncation), 2 u for the last factor and the store.  Instructions that add zeros round
nothing.  Two parts only would leave out up to 2^-14 of a product, typically 2^-16 = 256 u.

The smallest step of a bf16 value is 2^-133: what a value's three parts leave is below 2^-24 of it or below 2^-133, whichever is
more, and a product a b is off by up to 2^-133 (|a| + |b|) besides.  That counts where an operand is below about 2^-112, 2e-34."""
import numpy as np
import pytest
import torch

from distributed_tensorflow_amd.ops import vocab_head_bwd, vocab_head_fwd

gpu = pytest.mark.gpu
U = 2.0 ** -24


LEAST = 2.0 ** -133


def bound(terms, sums):
    """of a sum of products whose absolute values add up to ``sums``, ``terms`` of them not zero"""
    return (8 + 12 * terms + 2) * U * sums


# ------------------------------------------------------------------------------------- the bound tells parts apart
def parts(v, count, rounded=False):
    """The leading bits of ``v`` (fp32), cut ``count`` times to bf16; rounded: half a step added before the first cut."""
    left, out = v.astype(np.float32).copy(), []
    for q in range(count):
        half = np.uint32(0x8000 if rounded and q == 0 else 0)
        p = ((left.view(np.uint32) + half) & np.uint32(0xffff0000)).view(np.float32)
        out.append(p.astype(np.float64))
        left = (left - p).astype(np.float32)
    return out


TERMS = [(0, 2), (2, 0), (1, 1), (0, 1), (1, 0), (0, 0)]


def product(a, b, count=3, rounded=False, terms=TERMS):
    """a * b as the kernel forms it, summed in 64 bits"""
    pa, pb = parts(a, count, rounded), parts(b, count, rounded)
    return sum(pa[i] * pb[j] for i, j in terms if i < count and j < count)


@pytest.mark.parametrize("rounded", [False, True])
def test_three_parts_are_within_the_bound_and_less_is_not(rounded):
    g = np.random.default_rng(1)
    a, b = (g.standard_normal(100000).astype(np.float32) for _ in range(2))
    want = a.astype(np.float64) * b
    err = lambda x: np.abs(x - want) / np.abs(want)     # noqa: E731
    assert err(product(a, b, rounded=rounded)).max() <= 8 * U
    two = err(product(a, b, 2, rounded))
    assert np.median(two) > 2 * bound(1, 1.0) and (two > bound(1, 1.0)).mean() > 0.75
    # a term of the second order forgotten
    for lost in ((1, 1), (0, 2), (2, 0)):
        less = err(product(a, b, rounded=rounded, terms=[t for t in TERMS if t != lost]))
        assert (less > bound(1, 1.0)).mean() > 0.3, lost


@pytest.mark.parametrize("rounded", [False, True])
@pytest.mark.parametrize("exp", [-112, -120, -126, -132])
def test_small_values_keep_what_bf16_holds(exp, rounded):
    g = np.random.default_rng(2)
    a = (g.standard_normal(100000) * 2.0 ** exp).astype(np.float32)
    b = g.standard_normal(100000).astype(np.float32)
    want = a.astype(np.float64) * b
    d = np.abs(product(a, b, rounded=rounded) - want)
    assert (d <= 8 * U * np.abs(want) + LEAST * (np.abs(a.astype(np.float64)) + np.abs(b))).all()
    # only small values (a normal distribution has some of any size) lose more than others do
    more = d > 8 * U * np.abs(want)
    assert (np.abs(a[more].astype(np.float64)) < 2.0 ** -110).all() and (more.any() or exp == -112)


# --------------------------------------------------------------------------------------------------------- kernels
def within(got, want, limit, what):
    d = (got.double() - want).abs()
    assert bool((d <= limit).all()), f"{what}: {float((d / limit.clamp(min=1e-300)).max()):.3g} times its bound"


SHAPES = [(1, 300, 700, 0), (5, 600, 3001, 0), (40, 200, 777, 0), (64, 64, 5000, 256),         # dh and dw in 64-row tiles of four waves
          (100, 600, 3001, 0), (128, 2050, 300, 0), (100, 37, 1200, 512),                      # ... two by two
          (300, 600, 8003, 0), (700, 1000, 5011, 0), (1030, 2050, 1100, 0), (513, 33, 2049, 1024)]   # 128 x 128


@gpu
@pytest.mark.parametrize("n,hidden,classes,piece", SHAPES)
def test_gradients_of_single_products(gpu_lib, n, hidden, classes, piece):
    g = torch.Generator(device="cuda").manual_seed(n + hidden)
    h, w = (torch.randn((r, hidden), device="cuda", generator=g) for r in (n, classes))
    y = torch.randint(0, classes, (n,), device="cuda", generator=g)
    y[: min(n, 4)] = torch.tensor([classes - 1, 0, classes // 2, classes - 1], device="cuda")[: min(n, 4)]
    s = torch.rand(n, device="cuda", generator=g) + 0.5
    lse, bias = torch.full((n,), 1000.0, device="cuda"), torch.zeros(classes, device="cuda")
    dh, dw, db = vocab_head_bwd(h, w, y.to(torch.int32), lse, bias, row_scale=s, piece=piece)
    sd, hd, wd = s.double(), h.double(), w.double()
    want = -sd[:, None] * wd[y]
    within(dh, want, bound(1, want.abs()), "dh")
    each = sd[:, None] * hd
    zero = torch.zeros((classes, hidden), dtype=torch.float64, device="cuda")
    terms = torch.bincount(y, minlength=classes).double()[:, None]
    within(dw, zero.index_add(0, y, -each), bound(terms, zero.index_add(0, y, each.abs())), "dw")
    assert bool((dw[terms[:, 0] == 0] == 0).all())
    db_want = torch.zeros(classes, dtype=torch.float64, device="cuda").index_add(0, y, -sd)
    within(db, db_want, terms[:, 0] * U * db_want.abs(), "db")


@gpu
@pytest.mark.parametrize("n,hidden,classes", [(1, 300, 700), (5, 600, 3001), (40, 200, 777), (100, 1024, 10000), (300, 2048, 600), (300, 600, 8003),
                                              (1030, 520, 12001), (777, 64, 50001)])
def test_logits_of_single_products(gpu_lib, n, hidden, classes):
    """Rows with one value each, one class that is not masked: its log-sum-exp is one product.  Joining adds 4 u (1 + |z|)."""
    g = torch.Generator(device="cuda").manual_seed(n)
    w = torch.randn((classes, hidden), device="cuda", generator=g)
    k = torch.randint(0, hidden, (n,), device="cuda", generator=g)
    v = torch.rand(n, device="cuda", generator=g) + 0.5
    h = torch.zeros((n, hidden), device="cuda")
    h[torch.arange(n, device="cuda"), k] = v
    for c in (0, classes // 3, classes - 1):
        bias = torch.full((classes,), -torch.inf, device="cuda")
        bias[c] = 0.0
        y = torch.full((n,), c, dtype=torch.int32, device="cuda")
        loss, lse = vocab_head_fwd(h, w, y, bias)
        want = v.double() * w[c].double()[k]
        within(lse, want, bound(1, want.abs()) + 4 * U * (1 + want.abs()), f"lse of class {c}")
        assert float(loss.abs().max()) <= 4 * U * (1 + float(want.abs().max()))


@gpu
@pytest.mark.parametrize("exp", [-100, -112, -120, -126])
@pytest.mark.parametrize("n,hidden,classes", [(5, 200, 777), (100, 200, 777), (300, 200, 777)])
def test_small_upstream_gradients(gpu_lib, n, hidden, classes, exp):
    """row_scale is multiplied into d before d is cut into parts; grad_scale is not."""
    g = torch.Generator(device="cuda").manual_seed(n)
    h, w = (torch.randn((r, hidden), device="cuda", generator=g) for r in (n, classes))
    y = torch.randperm(classes, device="cuda", generator=g)[:n]
    lse = torch.full((n,), 1000.0, device="cuda")
    base = torch.rand(n, device="cuda", generator=g) + 0.5
    for s, grad_scale, least in ((base * 2.0 ** exp, 1.0, LEAST), (base, 2.0 ** exp, 0.0)):
        dh, dw, _ = vocab_head_bwd(h, w, y.to(torch.int32), lse, row_scale=s, grad_scale=grad_scale)
        sd = (s.double() * grad_scale)[:, None]
        for got, x, what in ((dh, w.double()[y], "dh"), (dw[y], h.double(), "dw")):
            want = -sd * x
            within(got, want, bound(1, want.abs()) + least * (sd + x.abs()) + 2.0 ** -149, what)
