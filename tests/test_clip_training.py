"""Gradient clipping inside training: HipEngine(clip_norm=...), the CPU oracle, --clip_norm, and a training step made of the
many-class head, the clipped gradients and the package's update kernel.

An SGD update w' = fma(-(lr f), g, w) is off by one rounding of w' (2^-24 |w'|) and three of lr f g (lr, f and their product)."""
import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from distributed_tensorflow_amd.models.oracle import OracleModel
from distributed_tensorflow_amd.models.spec import ModelSpec
from distributed_tensorflow_amd.ops import reference as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
gpu = pytest.mark.gpu
U = 2.0 ** -24


def norm_of(arena, layout, scale=1.0):
    return float(R.global_norm([layout.view(arena, n) for n in layout.names()], scale))


# ------------------------------------------------------------------------------------------------------------------ CPU
@pytest.mark.parametrize("optimizer", ["sgd", "adam"])
def test_oracle_clips_the_scaled_gradient(optimizer):
    spec = ModelSpec()
    g = torch.randn(OracleModel(spec).layout.total, generator=torch.Generator().manual_seed(1)) * 1e-3
    limit = 0.1
    a = OracleModel(spec, optimizer=optimizer, learning_rate=0.01, clip_norm=limit, seed=3)
    b = OracleModel(spec, optimizer=optimizer, learning_rate=0.01, seed=3)
    norm = norm_of(g, a.layout, 0.5)
    assert norm > limit
    a.apply_gradients(g, scale=0.5)
    b.apply_gradients(g, scale=0.5 * limit / norm)
    assert float(a.grad_norm) == pytest.approx(norm, rel=1e-6)
    for n in a.layout.names():
        # (Adam's first step is lr g / |g|: only its rounding differs)
        assert torch.allclose(a.params[n], b.params[n], rtol=1e-6, atol=1e-6)
    a.clip_norm = 2 * norm
    c = OracleModel(spec, optimizer=optimizer, learning_rate=0.01, seed=3)
    d = OracleModel(spec, optimizer=optimizer, learning_rate=0.01, clip_norm=2 * norm, seed=3)
    c.apply_gradients(g)
    d.apply_gradients(g)
    assert torch.equal(c.arena[:c.layout.ctrl], d.arena[:d.layout.ctrl])


def run_cli(args, ok=True):
    r = subprocess.run([sys.executable, os.path.join(ROOT, "mnistdist.py"), "--backend=cpu", "--synthetic", "--noeval", *args],
                       capture_output=True, text=True, cwd=ROOT, timeout=240, env=dict(os.environ, OMP_NUM_THREADS="2"))
    assert (r.returncode == 0) == ok, r.stdout + r.stderr
    return r.stdout + r.stderr


def test_cli_refuses_what_cannot_be_clipped():
    two = ["--job_name=worker", "--ps_hosts=127.0.0.1:1", "--worker_hosts=127.0.0.1:2,127.0.0.1:3", "--clip_norm=1"]
    assert "--clip_norm must be" in run_cli(["--clip_norm=-1"], ok=False)
    assert "--clip_norm must be" in run_cli(["--clip_norm=inf"], ok=False)
    assert "--clip_norm needs --mode=sync" in run_cli(two + ["--mode=async"], ok=False)
    assert "not with --p2p_allreduce" in run_cli(two + ["--mode=sync", "--p2p_allreduce"], ok=False)
    assert "not with --p2p_allreduce" in run_cli(two + ["--mode=sync", "--dense_update=sharded"], ok=False)


def check_step_length(p1, p2, lr, limit):
    """Plain SGD with a gradient that is longer than the limit moves the parameters by lr * limit."""
    d = float(np.linalg.norm(p2.astype(np.float64) - p1.astype(np.float64)))
    assert abs(d - lr * limit) <= 2 * U * float(np.linalg.norm(p2.astype(np.float64))) + 8 * U * lr * limit


def test_cli_clips_on_one_task(tmp_path):
    lr, limit, p = 0.01, 0.5, []
    for steps in (1, 2):
        f = tmp_path / f"p{steps}.npy"
        run_cli([f"--steps={steps}", "--batch_size=32", f"--learning_rate={lr}", f"--clip_norm={limit}", "--logdir=", f"--dump_params={f}"])
        p.append(np.load(f))
    check_step_length(p[0], p[1], lr, limit)


def test_cli_clips_the_mean_of_two_workers(tmp_path):
    sys.path.insert(0, os.path.join(ROOT, "tests"))
    from test_distributed_cpu import launch
    lr, limit, p = 0.01, 0.5, {}
    for steps in (1, 2):
        files = [str(tmp_path / f"w{i}_{steps}.npy") for i in range(2)]
        out = launch(1, 2, ["--mode=sync", "--batch_size=16", f"--steps={steps}", f"--learning_rate={lr}", f"--clip_norm={limit}",
                            "--noeval"], str(tmp_path / f"logs{steps}"),
                     per_task_extra={("worker", i): [f"--dump_params={files[i]}"] for i in range(2)})
        for key, (rc, o) in out.items():
            assert rc == 0, (key, o)
        p[steps] = [np.load(f) for f in files]
        spec_total = p[steps][0].size - 4                     # (the control block is no parameter)
        assert np.array_equal(p[steps][0][:spec_total], p[steps][1][:spec_total])
    check_step_length(p[1][0][:-4], p[2][0][:-4], lr, limit)


# ------------------------------------------------------------------------------------------------------------------ GPU
def make_engine(dtype="bf16", clip=0.0, optimizer="sgd", B=100, **kw):
    from distributed_tensorflow_amd.engine import DeviceDataset, HipEngine
    ds = DeviceDataset.synthetic(2048, seed=7, dtype=dtype)
    eng = HipEngine(ModelSpec(), B, ds, optimizer=optimizer, learning_rate=0.01, seed=5, dtype=dtype, clip_norm=clip, **kw)
    eng.init_params()
    return eng


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("multi_stream", [False, True])
def test_engine_applies_the_clipped_gradient(gpu_lib, dtype, multi_stream):
    limit = 0.3
    if dtype == "fp32" and multi_stream:
        pytest.skip("the fp32 kernels run on one stream")
    eng = make_engine(dtype, limit, multi_stream=multi_stream)
    eng.set_grad_scale(0.5)
    for step in range(3):
        before = eng.params.double().clone()
        eng.launch_train_step()
        norm = norm_of(eng.grads, eng.layout, 0.5)            # the arena keeps the unclipped gradient
        assert norm > limit and abs(eng.grad_norm() - norm) <= norm * (U + eng.layout.total * 2.0 ** -53)
        for n in eng.layout.names():
            w, g = eng.layout.view(before, n), eng.layout.view(eng.grads, n).double()
            move = 0.01 * 0.5 * (limit / norm) * g
            want = w - move
            d = (eng.layout.view(eng.params, n).double() - want).abs()
            # (0.01 itself is a float in device memory: one more rounding)
            assert bool((d <= U * want.abs() + 5 * U * move.abs()).all()), n
        assert eng.global_step == step + 1


@gpu
@pytest.mark.parametrize("dtype,optimizer", [("bf16", "sgd"), ("bf16", "adam"), ("fp32", "sgd"), ("fp32", "adam")])
def test_a_norm_within_the_limit_changes_no_bit(gpu_lib, dtype, optimizer):
    a, b = make_engine(dtype, 1e6, optimizer), make_engine(dtype, 0.0, optimizer)
    for _ in range(4):
        a.launch_train_step()
        b.launch_train_step()
    assert torch.equal(a.params[:a.layout.ctrl], b.params[:b.layout.ctrl]) and a.grad_norm() > 0
    with pytest.raises(RuntimeError, match="clip_norm > 0"):
        b.grad_norm()


@gpu
@pytest.mark.parametrize("optimizer", ["sgd", "adam"])
def test_replayed_steps_are_the_eager_ones(gpu_lib, optimizer):
    """The clipping factor is computed anew in every replay, and a changed learning rate reaches it."""
    a, b = make_engine("bf16", 0.2, optimizer), make_engine("bf16", 0.2, optimizer)
    a.capture()
    norms = []
    for step in range(5):
        if step == 3:
            a.set_learning_rate(0.002)
            b.set_learning_rate(0.002)
        a.train_step()
        b.launch_train_step()
        norms.append((a.grad_norm(), b.grad_norm()))
        assert torch.equal(a.params, b.params), step
    assert all(x == y for x, y in norms) and len({x for x, _ in norms}) == 5


@gpu
def test_the_explicit_batch_path_clips(gpu_lib):
    limit = 0.25
    a, b = make_engine("fp32", limit), make_engine("fp32", 0.0)
    x, y = a.dataset.images[:100].contiguous(), a.dataset.labels[:100].contiguous()
    before = a.params.double().clone()
    a.train_step_on(x, y)
    norm = norm_of(a.grads, a.layout)
    assert norm > limit and abs(a.grad_norm() - norm) <= norm * (U + a.layout.total * 2.0 ** -53)
    b.set_grad_scale(limit / norm)
    b.train_step_on(x, y)
    for n in a.layout.names():
        move = (a.layout.view(a.params, n).double() - a.layout.view(before, n)).abs()
        d = (a.layout.view(a.params, n) - b.layout.view(b.params, n)).abs().double()
        assert bool((d <= 2 * U * a.layout.view(a.params, n).abs().double() + 8 * U * move).all()), n


@gpu
def test_refusals(gpu_lib):
    for bad in (-1.0, math.nan, math.inf):
        with pytest.raises(ValueError, match="clip_norm"):
            make_engine(clip=bad)
    import ctypes
    eng = make_engine("bf16", 1.0)
    s = torch.cuda.current_stream().cuda_stream
    assert eng.lib.dtf_engine_dp_phase1(eng._d(), 0, s, s) == -1          # the overlapped data-parallel schedule
    assert eng.lib.dtf_engine_dp_step(eng._d(), None, 1, 1, s, s) == -1
    del ctypes


@gpu
def test_a_gradient_that_is_not_finite_is_loud(gpu_lib):
    eng = make_engine("fp32", 1.0)
    eng.launch_train_step()
    eng.grads[123] = math.nan
    eng.launch_update()
    assert math.isnan(eng.grad_norm()) and bool(torch.isnan(eng.params[:eng.layout.sizes["wd1"]]).all())


# -------------------------------------------------------------------------------- head, clipping and update together
class HeadTrainer:
    """A linear classifier over many classes, trained with the package's kernels: fp32 master weights and gradients in flat
    arenas, a bf16 copy of the weight for the products."""

    def __init__(self, hidden, classes, lr, limit, seed=0):
        from distributed_tensorflow_amd.ops import GlobalNormClip, native
        self.lib, self.hidden, self.classes, self.limit = native.load(), hidden, classes, limit
        g = torch.Generator(device="cuda").manual_seed(seed)
        n = hidden * classes
        self.n = n + (-(-classes // 4)) * 4
        self.params = torch.zeros(self.n, device="cuda")
        self.params[:n] = torch.randn(n, device="cuda", generator=g) * 0.1
        self.grads = torch.zeros_like(self.params)
        self.shadow = self.params.bfloat16()
        self.hyper = torch.tensor([lr, 0.9, 0.999, 1e-8, 1.0, 0, 0, 0, 0, 0, 0, 0], device="cuda")
        self.wT, self.bias = self.shadow[:n].view(classes, hidden), self.params[n:n + classes]
        self.dwT, self.dbias = self.grads[:n].view(classes, hidden), self.grads[n:n + classes]
        self.clip = GlobalNormClip([self.dwT, self.dbias])

    def step(self, h, labels):
        from distributed_tensorflow_amd.ops import vocab_head_bwd, vocab_head_fwd
        from distributed_tensorflow_amd.ops.native import check, ptr
        loss, lse = vocab_head_fwd(h, self.wT, labels, self.bias)
        dh, _, _ = vocab_head_bwd(h, self.wT, labels, lse, self.bias, grad_scale=1.0 / h.shape[0], dwT=self.dwT, dbias=self.dbias)
        _, norm = self.clip.clip(self.limit)
        check(self.lib.dtf_sgd_update(ptr(self.params), ptr(self.grads), ptr(self.shadow), ptr(self.hyper), self.n, None, 0, 0, 0,
                                      torch.cuda.current_stream().cuda_stream), "sgd_update")
        return loss, dh, norm


@gpu
def test_head_clip_and_update_make_a_training_step(gpu_lib):
    n, hidden, classes, lr, limit = 200, 64, 1001, 0.5, 0.05
    g = torch.Generator(device="cuda").manual_seed(2)
    h = torch.randn((n, hidden), device="cuda", generator=g).bfloat16()
    labels = torch.randint(0, classes, (n,), device="cuda", generator=g, dtype=torch.int32)
    labels[5] = -1
    t = HeadTrainer(hidden, classes, lr, limit)
    w0, b0, p0 = t.wT.double().clone(), t.bias.double().clone(), t.params.double().clone()
    loss, dh, norm = t.step(h, labels)
    # the same step in 64 bits, through autograd; the bounds of the head's results are those of its own tests
    from test_vocab_head import Exact, within
    w, b = w0.clone().requires_grad_(True), b0.clone().requires_grad_(True)
    z = h.double() @ w.t() + b
    ref = torch.nn.functional.cross_entropy(z, labels.long(), ignore_index=-1, reduction="none")
    (ref.sum() / n).backward()
    x = Exact(h, w0.bfloat16(), labels, b0.float(), grad_scale=1.0 / n)
    (_, dw_bound), (_, db_bound) = x.dw(torch.float32), x.db()
    within(loss, ref.detach(), x.e_loss, "loss")
    within(dh, *x.dh(), "dh")
    assert float(loss[5]) == 0.0
    ref_norm = math.sqrt(float(w.grad.square().sum() + b.grad.square().sum()))
    off = math.sqrt(float(dw_bound.square().sum() + db_bound.square().sum()))      # | |a| - |b| | <= |a - b|
    assert ref_norm > limit and abs(float(norm) - ref_norm) <= off + U * ref_norm
    # what was applied: the clipped gradients in the arena, whose norm is the limit
    assert abs(math.sqrt(float(t.grads.double().square().sum())) - limit) <= limit * 4 * U
    moved = p0 - t.params.double()
    assert bool(((moved - lr * t.grads.double()).abs() <= U * t.params.double().abs() + 4 * U * lr * t.grads.double().abs()).all())
    assert torch.equal(t.shadow, t.params.bfloat16())
    factor = limit / ref_norm
    slack = off / ref_norm + 4 * U                                                 # of the factor
    within(t.dwT, w.grad * factor, (dw_bound + w.grad.abs() * slack) * factor * (1 + slack), "clipped dw")
    within(t.dbias, b.grad * factor, (db_bound + b.grad.abs() * slack) * factor * (1 + slack), "clipped db")


@gpu
def test_head_training_steps_replay_as_a_graph(gpu_lib):
    n, hidden, classes = 130, 40, 700
    g = torch.Generator(device="cuda").manual_seed(4)
    batches = [((torch.randn((n, hidden), device="cuda", generator=g)).bfloat16(),
                torch.randint(0, classes, (n,), device="cuda", generator=g, dtype=torch.int32)) for _ in range(4)]
    a, b = HeadTrainer(hidden, classes, 0.5, 0.05, seed=1), HeadTrainer(hidden, classes, 0.5, 0.05, seed=1)
    h, y = batches[0][0].clone(), batches[0][1].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, _, norm = a.step(h, y)
    for hb, yb in batches:
        h.copy_(hb)
        y.copy_(yb)
        graph.replay()
        want_loss, _, want_norm = b.step(hb, yb)
        torch.cuda.synchronize()
        assert torch.equal(loss, want_loss) and torch.equal(norm, want_norm) and torch.equal(a.params, b.params)
