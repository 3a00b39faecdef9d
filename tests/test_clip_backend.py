"""Gradient clipping through the HIP backend as the trainer builds it (fused dense update, graph replay above 1024 images), and
through the command line on a GPU: one task, and two synchronous workers that share the device.

Plain SGD with a gradient longer than the limit moves the parameters by lr * limit.  w' = fma(-(lr f), g, w) is off by one
rounding of w' and three of lr f g."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from distributed_tensorflow_amd.models.spec import ModelSpec
from distributed_tensorflow_amd.ops import reference as R
from test_clip_training import check_step_length

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
U = 2.0 ** -24
LR, LIMIT = 0.01, 0.3


def make(dtype="bf16", clip=LIMIT, batch=100, optimizer="sgd"):
    from distributed_tensorflow_amd.backends import HipBackend
    from distributed_tensorflow_amd.data.mnist import read_data_sets
    data = read_data_sets("", synthetic=True, synthetic_sizes=(4096, 256))
    b = HipBackend(ModelSpec(), batch, data, optimizer=optimizer, learning_rate=LR, seed=3, dtype=dtype, clip_norm=clip)
    b.init_params(5)
    return b


def check_move(b, before, scale):
    """every element, from the gradient in the arena"""
    eng, lay = b.engine, b.layout
    norm = float(R.global_norm([lay.view(eng.grads, n) for n in lay.names()], scale))
    assert norm > LIMIT and abs(eng.grad_norm() - norm) <= norm * (U + lay.total * 2.0 ** -53)
    for n in lay.names():
        move = LR * scale * (LIMIT / norm) * lay.view(eng.grads, n).double()
        want = lay.view(before, n) - move
        d = (lay.view(eng.params, n).double() - want).abs()
        assert bool((d <= U * want.abs() + 5 * U * move.abs()).all()), n


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_local_steps_of_the_backend(gpu_lib, dtype):
    b = make(dtype)
    assert b.clip_norm == LIMIT and b.engine.fuse_dense_update
    for step in range(3):
        before = b.params.double().clone()
        b.train_step_local()
        check_move(b, before, 1.0)
        assert b.get_global_step() == step + 1


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_gradients_computed_and_applied_apart(gpu_lib, dtype):
    """What a synchronous worker does, with the mean of two equal gradients."""
    b = make(dtype)
    for _ in range(2):
        before = b.params.double().clone()
        b.compute_gradients()
        b.grads.mul_(2.0)
        b.apply_gradients(scale=0.5)
        check_move(b, before, 0.5)


@pytest.mark.parametrize("optimizer", ["sgd", "adam"])
def test_replayed_steps_of_a_large_batch(gpu_lib, optimizer):
    a, b = make(batch=1152, optimizer=optimizer), make(batch=1152, optimizer=optimizer)
    assert a.use_graph
    b.use_graph = False
    for step in range(4):
        a.train_step_local()
        b.train_step_local()
        assert torch.equal(a.params, b.params) and a.engine.grad_norm() == b.engine.grad_norm() > LIMIT, step


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_cli_clips_on_one_task(gpu_lib, tmp_path, dtype):
    p = []
    for steps in (1, 2):
        f = tmp_path / f"p{steps}.npy"
        r = subprocess.run([sys.executable, os.path.join(ROOT, "mnistdist.py"), "--backend=hip", "--synthetic", "--noeval", f"--steps={steps}",
                            "--batch_size=64", f"--learning_rate={LR}", f"--clip_norm={LIMIT}", f"--dtype={dtype}", "--logdir=",
                            f"--dump_params={f}"], capture_output=True, text=True, cwd=ROOT, timeout=100)
        assert r.returncode == 0, r.stdout + r.stderr
        p.append(np.load(f))
    check_step_length(p[0], p[1], LR, LIMIT)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_cli_clips_the_mean_of_two_workers(gpu_lib, tmp_path, dtype):
    from test_distributed_cpu import launch
    p = {}
    for steps in (1, 2):
        files = [str(tmp_path / f"w{i}_{steps}.npy") for i in range(2)]
        out = launch(1, 2, ["--mode=sync", "--comm_backend=gloo", "--batch_size=64", f"--steps={steps}", f"--learning_rate={LR}",
                            f"--clip_norm={LIMIT}", f"--dtype={dtype}", "--noeval"], str(tmp_path / f"logs{steps}"), timeout=100,
                     backend="hip", per_task_extra={("worker", i): [f"--dump_params={files[i]}"] for i in range(2)})
        for key, (rc, o) in out.items():
            assert rc == 0, (key, o[-3000:])
        p[steps] = [np.load(f) for f in files]
        assert np.array_equal(p[steps][0][:-4], p[steps][1][:-4]), "the replicas differ"
    check_step_length(p[1][0][:-4], p[2][0][:-4], LR, LIMIT)
