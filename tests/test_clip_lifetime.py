"""How long the memory of a GlobalNormClip lives (ops/clip.py).

The kernels read the plan's table and walk the addresses in it.  PyTorch's allocator hands a block out again, on the stream it
was allocated on, as soon as its last tensor is gone, whatever another stream still does with it -- unless that stream was
recorded for the block.  A plan that is made on one stream, used on another and dropped has to record it."""
import math

import pytest
import torch

from distributed_tensorflow_amd.ops import GlobalNormClip, clip

gpu = pytest.mark.gpu


class Recorder:
    """Stands for a tensor; notes the streams it is recorded for."""

    def __init__(self):
        self.streams = []

    def record_stream(self, s):
        self.streams.append(s)

    def data_ptr(self):
        return 0


class Lib:
    def dtf_global_norm(self, *a):
        return 0

    def dtf_clip_by_global_norm(self, *a):
        return 0


@pytest.fixture
def plan(monkeypatch):
    """A plan made on stream 7, without a GPU; ``now``: the stream of a call, whether it is captured."""
    now = dict(stream=7, capturing=False)

    class OnDevice:
        def __init__(self, device):
            pass

        def __enter__(self):
            return now["stream"]

        def __exit__(self, *_):
            pass

    monkeypatch.setattr(clip, "on_device", OnDevice)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now["capturing"])
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: now["stream"])
    p = object.__new__(GlobalNormClip)
    p.device, p.lib, p.table, p.chunks, p.slots, p.out = torch.device("cpu"), Lib(), Recorder(), 1, 1, []
    p._in_place, p._clip_error, p._streams = 1, None, {7}
    p._memory = [p.table, Recorder(), Recorder()]
    return p, now


@pytest.mark.parametrize("call", [lambda p: p.norm(), lambda p: p.clip(1.0)])
def test_a_call_on_another_stream_is_recorded(plan, call):
    p, now = plan
    call(p)
    assert all(m.streams == [] for m in p._memory)          # the plan's own stream: freed memory follows its work anyway
    now["stream"] = 9
    call(p)
    call(p)
    assert all(m.streams == [9] for m in p._memory)         # once is enough: the allocator looks when the block is freed
    now["stream"] = 11
    call(p)
    now["stream"] = 9
    call(p)
    assert all(m.streams == [9, 11] for m in p._memory)


def test_a_captured_call_is_not_recorded(plan):
    """The graph's replays, not the captured call, read the table: whoever keeps the graph keeps the plan."""
    p, now = plan
    now.update(stream=9, capturing=True)
    p.norm()
    assert all(m.streams == [] for m in p._memory)
    now["capturing"] = False
    p.norm()
    assert all(m.streams == [9] for m in p._memory)


def test_the_list_of_outputs_is_the_callers(plan):
    """What a caller does to the list that a call returned must not change the next call's."""
    p, _ = plan
    a, b = torch.zeros(1), torch.zeros(1)
    p.out = [a, b]
    got, _ = p.clip(1.0)
    assert got[0] is a and got[1] is b
    got.clear()
    assert len(p.clip(1.0)[0]) == 2


@gpu
def test_memory_of_a_dropped_plan_is_not_handed_out_while_it_is_read(gpu_lib):
    """The call waits on its stream behind other work; the plan and its tensors are gone before it runs."""
    made, used = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(made):
        tensors = [torch.full((3000 + k,), 0.5, device="cuda") for k in range(3)]
        out = [torch.empty_like(t) for t in tensors]
        plan = GlobalNormClip(tensors, out=out)
    torch.cuda.synchronize()
    want = math.sqrt(0.25 * sum(t.numel() for t in tensors))
    taken = {t.untyped_storage().data_ptr() for t in tensors + out + [plan.table]}
    sizes = [t.untyped_storage().nbytes() for t in tensors + out + [plan.table]]
    with torch.cuda.stream(used):
        torch.cuda._sleep(200_000_000)
        norm = plan.norm()
    assert not used.query()                                  # (the work before it is still running)
    del plan, tensors, out
    with torch.cuda.stream(made):
        fresh = [torch.zeros(n, dtype=torch.uint8, device="cuda") for n in sizes]
    assert not taken & {t.untyped_storage().data_ptr() for t in fresh}
    torch.cuda.synchronize()
    assert abs(float(norm) - want) <= want * 2.0 ** -23
