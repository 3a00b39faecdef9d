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
