"""vocab_head_bwd(keep_rounding=True): the logits' gradient d of bf16 operands as two bf16 values, for any number of rows.

d = d1 + d2 is off by half a step of half a step (2^-16 of d), whatever the row; the bounds are test_vocab_head.py's with that in
the place of d's own rounding.  Every product is formed twice, so the running sums have twice the terms."""
import math

import pytest
import torch

from distributed_tensorflow_amd.ops import vocab_head_bwd, vocab_head_fwd
from test_vocab_head import Exact, U, make, within, without_own_rounding

gpu = pytest.mark.gpu


def check(h, w, y, b, s=1.0, row_scale=None, piece=0):
    x = Exact(h, w, y, b, grad_scale=s, row_scale=row_scale)
    _, lse = vocab_head_fwd(h, w, y, b)
    dw = torch.full(w.shape, 9.0, device="cuda")
    dh, _, db = vocab_head_bwd(h, w, y, lse, b, grad_scale=s, row_scale=row_scale, dwT=dw, piece=piece, keep_rounding=True)
    within(dw, *without_own_rounding(x, s, True), "dw")
    got = x.d @ x.w
    e = (2 * x.e_d + (x.half ** 2 + 8 * math.sqrt(2 * w.shape[0]) * U) * x.d.abs()) @ x.w.abs()
    within(dh, got, e + x.half * (got.abs() + e), "dh")
    if b is not None:
        within(db, *x.db(), "db")
    return dh, dw, db, lse


SHAPES = [(33, 96, 400, 0), (64, 40, 1000, 256), (65, 200, 777, 0), (128, 33, 2100, 512),       # small tiles, weights read in place
          (129, 72, 513, 0), (300, 600, 8003, 0), (700, 1000, 5011, 2048), (777, 64, 50001, 0),  # 128 x 128; rounds and small tiles
          (1000, 40, 10007, 0), (1100, 1800, 3000, 0), (1030, 2050, 1100, 512), (1, 64, 300, 0), (17, 96, 1111, 256)]


@gpu
@pytest.mark.parametrize("n,hidden,classes,piece", SHAPES)
def test_against_the_formula(gpu_lib, n, hidden, classes, piece):
    h, w, y, b = make(n, hidden, classes, "bf16", bias=True, ignored=0.1 if n > 1 else 0.0, seed=n + classes)
    one = check(h, w, y, b, s=0.3, piece=piece)
    two = check(h, w, y, b, s=0.3, piece=piece)
    assert all(torch.equal(a, c) for a, c in zip(one, two))
    assert bool((one[0][y == -1] == 0).all())
    if n <= 32:         # kept anyway: the same bits
        dw = torch.empty_like(one[1])
        dh, _, db = vocab_head_bwd(h, w, y, one[3], b, grad_scale=0.3, dwT=dw, piece=piece)
        assert torch.equal(dh, one[0]) and torch.equal(dw, one[1]) and torch.equal(db, one[2])


@gpu
@pytest.mark.parametrize("n", [50, 300])
def test_what_it_is_for(gpu_lib, n):
    """Ordinary rows and an fp32 gradient of the weight: d's rounding, up to 2^-8 of a value, shows in it, and is gone."""
    h, w, y, _ = make(n, 64, 3000, "bf16", seed=n)
    x = Exact(h, w, y)
    _, lse = vocab_head_fwd(h, w, y)
    rms = []
    for keep in (False, True):
        dw = torch.empty(w.shape, device="cuda")
        dh, _, _ = vocab_head_bwd(h, w, y, lse, dwT=dw, keep_rounding=keep)
        want = x.d.t() @ x.h
        rms.append(float((dw.double() - want).square().mean().sqrt() / want.square().mean().sqrt()))
    assert rms[1] < rms[0] / 30, rms


@gpu
def test_row_scales_and_strided_rows(gpu_lib):
    h, w, y, b = make(140, 96, 900, "bf16", bias=True, ignored=0.2, seed=3)
    scale = torch.rand(140, device="cuda") + 0.1
    scale[5] = 0.0
    base = check(h, w, y, b, s=0.25, row_scale=scale)
    big_h, big_w = (torch.full((t.shape[0], 103), math.nan, device="cuda").bfloat16() for t in (h, w))
    big_h[:, 3:99], big_w[:, 3:99] = h, w
    again = check(big_h[:, 3:99], big_w[:, 3:99], y, b, s=0.25, row_scale=scale)
    assert all(torch.equal(a, c) for a, c in zip(base, again))


@gpu
def test_fp32_operands_have_nothing_to_keep(gpu_lib):
    h, w, y, b = make(140, 96, 900, "fp32", bias=True, seed=4)
    _, lse = vocab_head_fwd(h, w, y, b)
    a, c = (vocab_head_bwd(h, w, y, lse, b, keep_rounding=k) for k in (False, True))
    assert all(torch.equal(x, z) for x, z in zip(a, c))


@gpu
@pytest.mark.parametrize("n", [40, 300])
def test_one_of_the_gradients_alone_and_replayed(gpu_lib, n):
    h, w, y, b = make(n, 72, 2100, "bf16", bias=True, ignored=0.1, seed=5)
    _, lse = vocab_head_fwd(h, w, y, b)
    dh, dw, db = vocab_head_bwd(h, w, y, lse, b, keep_rounding=True)
    only_h = vocab_head_bwd(h, w, y, lse, b, keep_rounding=True, need_dwT=False)
    only_w = vocab_head_bwd(h, w, y, lse, b, keep_rounding=True, need_dh=False)
    assert torch.equal(only_h[0], dh) and torch.equal(only_w[1], dw) and only_h[1] is None and only_w[0] is None
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = vocab_head_bwd(h, w, y, lse, b, keep_rounding=True, piece=512)
    for rep in range(3):
        for t, f in zip((h, w, y, b), make(n, 72, 2100, "bf16", bias=True, ignored=0.1, seed=40 + rep)):
            t.copy_(f)
        lse.copy_(vocab_head_fwd(h, w, y, b)[1])
        want = vocab_head_bwd(h, w, y, lse, b, keep_rounding=True, piece=512)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(got, want)), rep


def test_workspace_counts_the_second_rows():
    """Host code: what is kept needs twice the rows, and nothing where it is kept anyway or has no place."""
    from distributed_tensorflow_amd.ops import native
    lib = native.load()

    def need(kind, n, dt=1):
        return lib.dtf_vocab_head_workspace(dt, kind, 1 << 20, 512, 1 << 30, 512, n, 512, 4096, 0, 0)

    d, h = 300 * 4096 * 2, 300 * 512 * 2
    assert need(2, 300) >= need(1, 300) + d + h - 1024
    assert need(2, 32) == need(1, 32) and need(2, 300, 0) == need(1, 300, 0)
    assert need(3, 300) == -3 and need(-1, 300) == -3
