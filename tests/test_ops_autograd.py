"""The head and the clipping next to PyTorch's autograd: they record nothing, so under grad mode operands that require gradients
are refused, and what they write in place counts as written (a backward pass that saved it must not use it)."""
import pytest
import torch

from distributed_tensorflow_amd.ops import GlobalNormClip, vocab_head_bwd, vocab_head_fwd

gpu = pytest.mark.gpu


def operands(device="cpu"):
    g = torch.Generator().manual_seed(1)
    h, w, b = torch.randn(4, 8, generator=g), torch.randn(16, 8, generator=g), torch.randn(16, generator=g)
    return [t.to(device) for t in (h, w)] + [torch.tensor([1, 0, 15, 7], dtype=torch.int32, device=device), b.to(device)]


@pytest.mark.parametrize("which", [0, 1, 3])
def test_the_head_refuses_operands_that_require_gradients(which):
    a = operands()
    a[which].requires_grad_(True)
    with pytest.raises(ValueError, match="require gradients"):
        vocab_head_fwd(*a)
    lse = torch.zeros(4)
    with pytest.raises(ValueError, match="require gradients"):
        vocab_head_bwd(a[0], a[1], a[2], lse, a[3])
    with torch.no_grad(), pytest.raises(ValueError, match="GPU tensors expected"):
        vocab_head_fwd(*a)
    with pytest.raises(ValueError, match="GPU tensors expected"):
        vocab_head_fwd(*(t.detach() for t in a))


@pytest.mark.parametrize("name", ["row_scale", "dh", "dwT", "dbias"])
def test_the_backward_pass_refuses_the_others_too(name):
    h, w, y, b = operands()
    t = dict(row_scale=torch.ones(4), dh=torch.zeros(4, 8), dwT=torch.zeros(16, 8), dbias=torch.zeros(16))[name].requires_grad_(True)
    with pytest.raises(ValueError, match="require gradients"):
        vocab_head_bwd(h, w, y, torch.zeros(4), b, **{name: t})


def test_a_plan_refuses_tensors_that_require_gradients():
    x = torch.zeros(8)
    p = torch.zeros(8, requires_grad=True)
    for args in (dict(tensors=[x, p]), dict(tensors=[x], out=[p])):
        with pytest.raises(ValueError, match="require gradients"):
            GlobalNormClip(**args)
        with torch.no_grad(), pytest.raises(ValueError, match="GPU tensors expected"):
            GlobalNormClip(**args)


@gpu
def test_parameters_under_no_grad(gpu_lib):
    h, w, y, b = operands("cuda")
    want = vocab_head_fwd(h, w, y, b)
    for t in (h, w, b):
        t.requires_grad_(True)
    with torch.no_grad():
        loss, lse = vocab_head_fwd(h, w, y, b)
        grads = vocab_head_bwd(h, w, y, lse, b)
        plan = GlobalNormClip([h, w])
        norm = plan.norm()
    assert torch.equal(loss, want[0]) and all(not t.requires_grad for t in (loss, lse, norm) + grads)
    # the plan outlives the block it was made in
    with pytest.raises(ValueError, match="require gradients"):
        plan.norm()
    with pytest.raises(ValueError, match="require gradients"):
        plan.clip(1.0)


@gpu
def test_what_is_written_counts_as_written(gpu_lib):
    """Saved for a backward pass and then overwritten: autograd has to notice."""
    h, w, y, b = operands("cuda")
    _, lse = vocab_head_fwd(h, w, y, b)

    def saved(t):
        x = torch.ones_like(t, requires_grad=True)
        return (x * t).sum()        # keeps t for x's gradient

    dh, dw, db = torch.zeros_like(h), torch.zeros_like(w), torch.zeros_like(b)
    sums = [saved(t) for t in (dh, dw, db)]
    vocab_head_bwd(h, w, y, lse, b, dh=dh, dwT=dw, dbias=db)
    flat = torch.ones(100, device="cuda")
    views = list(torch.split(flat, [30, 70]))
    alone = torch.ones(5, device="cuda")
    sums += [saved(flat), saved(views[1]), saved(alone)]
    GlobalNormClip(views + [alone]).clip(1.0)
    out = [torch.zeros_like(t) for t in views]
    sums += [saved(t) for t in out]
    GlobalNormClip(views, out=out).clip(1.0)
    for s in sums:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            s.backward()
    # what is only read stays usable
    kept = saved(flat)
    GlobalNormClip(views).norm()
    GlobalNormClip(views, out=out).clip(1.0)
    kept.backward()


@gpu
def test_inference_tensors_have_no_counter(gpu_lib):
    with torch.inference_mode():
        t = torch.ones(100, device="cuda")
        GlobalNormClip([t]).clip(1.0)
        assert abs(float(t.double().norm()) - 1.0) <= 1e-6
