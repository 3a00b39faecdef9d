"""Where clipping by the global norm has no place, or was not asked for in the right order, an engine that clips says so."""
from types import SimpleNamespace

import pytest
import torch

from distributed_tensorflow_amd.backends import CpuBackend
from distributed_tensorflow_amd.cluster import ClusterSpec, TaskInfo
from distributed_tensorflow_amd.data.mnist import read_data_sets
from distributed_tensorflow_amd.models.spec import ModelSpec
from distributed_tensorflow_amd.parallel.async_push import AsyncPushServer, AsyncPushWorker
from distributed_tensorflow_amd.parallel.strategies import AsyncP2PServer, AsyncP2PWorker, AsyncRounds

CLUSTER = ClusterSpec({"ps": ["127.0.0.1:1"], "worker": ["127.0.0.1:2", "127.0.0.1:3"]})
PS, WORKER = TaskInfo(CLUSTER, "ps", 0), TaskInfo(CLUSTER, "worker", 0)


# ---------------------------------------------------------------------------------- the asynchronous strategies
def cpu_backend(clip_norm):
    data = read_data_sets("", synthetic=True, synthetic_sizes=(64, 16))
    return CpuBackend(ModelSpec(), 8, data, clip_norm=clip_norm)


@pytest.mark.parametrize("make", [lambda b: AsyncP2PServer(b, PS, 1, 10), lambda b: AsyncP2PWorker(b, WORKER, 1)])
def test_a_parameter_server_that_sees_shards_refuses_clipping(make):
    with pytest.raises(ValueError, match="no gradient clipping"):
        make(cpu_backend(1.0))
    make(cpu_backend(0.0))


@pytest.mark.parametrize("task", [PS, WORKER])
def test_a_parameter_server_that_sums_rounds_refuses_clipping(task):
    with pytest.raises(ValueError, match="no gradient clipping"):
        AsyncRounds(cpu_backend(1.0), task, 1)


@pytest.mark.parametrize("make", [lambda b: AsyncPushServer(b, PS, 1, 10), lambda b: AsyncPushWorker(b, WORKER, 1)])
def test_the_mailbox_parameter_server_refuses_clipping(make):
    """Before anything collective or native: no process group and no GPU here."""
    with pytest.raises(ValueError, match="no gradient clipping"):
        make(SimpleNamespace(name="hip", clip_norm=1.0, engine=SimpleNamespace(clip_norm=1.0)))


# ------------------------------------------------------------------------------------------- the engine's phases
class Lib:
    """Stands for the kernel library: every call succeeds and is noted."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *a: self.calls.append(name) or 0


@pytest.fixture
def engine(monkeypatch):
    from distributed_tensorflow_amd.engine import HipEngine
    monkeypatch.setattr(HipEngine, "_s", lambda self: 0)
    monkeypatch.setattr(HipEngine, "_d", lambda self: None)
    monkeypatch.setattr(HipEngine, "__del__", lambda self: None)
    eng = object.__new__(HipEngine)
    eng.lib, eng.clip_norm, eng.step_inc, eng.dtype, eng.dense_g16 = Lib(), 1.0, 1, "bf16", None
    eng.layout, eng.hyper, eng.B, eng._graph = SimpleNamespace(total=64), torch.zeros(12), 4, None
    return eng


X = torch.zeros(1)
NEW_GRADIENTS = [
    lambda e: e.launch_backward_dense(), lambda e: e.launch_backward_conv(X, None), lambda e: e.launch_backward(X, None),
    lambda e: e.launch_train_step(), lambda e: e.set_learning_rate(0.1), lambda e: e.set_grad_scale(0.5),
]


@pytest.mark.parametrize("k", range(len(NEW_GRADIENTS)))
def test_an_update_with_the_factor_of_another_gradient_is_refused(engine, k):
    """The clipping factor, the learning rate and the gradient scale of an update are those of the last launch_clip()."""
    with pytest.raises(RuntimeError, match=r"launch_clip\(\) first"):
        engine.launch_update_range(0, 64, True)             # no factor at all yet
    engine.launch_clip()
    engine.launch_update_range(0, 32, False)                # the ranges of one step share the factor
    engine.launch_update_range(32, 64, True)
    NEW_GRADIENTS[k](engine)
    done = len(engine.lib.calls)
    with pytest.raises(RuntimeError, match=r"launch_clip\(\) first"):
        engine.launch_update_range(0, 64, True)
    assert len(engine.lib.calls) == done                    # nothing was launched
    engine.launch_update()
    assert engine.lib.calls[done:done + 2] == ["dtf_engine_clip", "dtf_engine_update_range"]


def test_without_clipping_the_ranges_need_nothing(engine):
    engine.clip_norm = 0.0
    engine.launch_update_range(0, 64, True)
    engine.launch_backward_dense()
    engine.launch_update_range(0, 64, True)


def test_the_16_bit_dense_gradient_has_no_norm(engine):
    """With it the fc1 weight gradient never reaches the fp32 arena, whose norm is taken."""
    with pytest.raises(ValueError, match="no gradient clipping"):
        engine.enable_dense_g16()
    assert engine.dense_g16 is None
