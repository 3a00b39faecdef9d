"""Global norm and clipping (ops/clip.py, csrc/kernels/clip.hip) against 64-bit arithmetic.

Tolerances.  The norm is a sum of n non-negative fp64 terms (relative error at most n 2^-53, whatever the order), its root,
and one rounding to fp32.  A clipped value is g * f: f rounded once to fp32 and the product once more in fp32, then once to
the tensor's type (half a step; below the normal range of fp16 half of 2^-24)."""
import math

import pytest
import torch

from distributed_tensorflow_amd.ops import GlobalNormClip
from distributed_tensorflow_amd.ops import reference as R

DEV = "cuda"
gpu = pytest.mark.gpu


def norm_tol(tensors):
    return 2.0 ** -24 + sum(t.numel() for t in tensors) * 2.0 ** -53


def check_values(got, want64, dtype):
    half = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    tol = want64.abs() * (2 * 2.0 ** -24 + 2.0 ** -40 + half)
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25
    d = (got.double() - want64).abs()
    assert bool((d <= tol).all()), f"off by {float((d - tol).max()):.3g} beyond the bound"


def make(shapes, dtypes, seed=0, scale=1e-2):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [(torch.randn(s, device=DEV, generator=g) * scale).to(dt) for s, dt in zip(shapes, dtypes)]


def factor_of(norm, limit, scale=1.0):
    return scale * (limit / norm if norm > limit else 1.0)


# ------------------------------------------------------------------------------------------------ refusals (no GPU)
def test_refuses_what_it_cannot_walk():
    x = torch.zeros(8, 16)
    with pytest.raises(ValueError, match="no tensors"):
        GlobalNormClip([])
    with pytest.raises(TypeError, match="fp32, bf16 or fp16"):
        GlobalNormClip([x.double()])
    with pytest.raises(TypeError, match="strided"):
        GlobalNormClip([[1.0]])
    with pytest.raises(TypeError, match="strided"):
        GlobalNormClip([x.to_sparse()])
    with pytest.raises(ValueError, match="share memory"):
        GlobalNormClip([torch.zeros(1, 16).expand(8, 16)])
    with pytest.raises(ValueError, match="share memory"):
        GlobalNormClip([torch.as_strided(x, (3, 2), (1, 1))])
    with pytest.raises(ValueError, match="neither dense nor"):
        GlobalNormClip([x[::2, ::2]])
    with pytest.raises(ValueError, match="1 tensors but 2 outputs"):
        GlobalNormClip([x], out=[x, x])
    with pytest.raises(ValueError, match="shape and type"):
        GlobalNormClip([x], out=[torch.zeros(8, 15)])
    with pytest.raises(ValueError, match="shape and type"):
        GlobalNormClip([x], out=[x.bfloat16()])
    with pytest.raises(ValueError, match="an output shares memory"):
        GlobalNormClip([x, x.clone()], out=[torch.zeros(8, 16)] + [x])          # x is read as one, written as the other
    flat = torch.zeros(20)
    with pytest.raises(ValueError, match="an output shares memory"):
        GlobalNormClip([torch.zeros(10), torch.zeros(11)], out=[flat[:10], flat[9:]])
    with pytest.raises(ValueError, match="GPU tensors expected"):
        GlobalNormClip([x])


def test_reference_form():
    t = [torch.tensor([3.0, 0.0]), torch.tensor([[4.0]])]
    assert float(R.global_norm(t)) == 5.0
    out, norm = R.clip_by_global_norm(t, 2.5)
    assert float(norm) == 5.0 and torch.equal(out[0], torch.tensor([1.5, 0.0])) and torch.equal(out[1], torch.tensor([[2.0]]))
    out, _ = R.clip_by_global_norm(t, 5.0)
    assert torch.equal(out[0], t[0])
    out, norm = R.clip_by_global_norm([torch.tensor([1.0, math.inf])], 1.0)
    assert bool(torch.isnan(out[0]).all())


# ----------------------------------------------------------------------------------------------------------- values
F, B, H = torch.float32, torch.bfloat16, torch.float16
LISTS = [
    ([(1,)], [F]),
    ([()], [B]),
    ([(0,), (5,), (0, 3)], [B, F, H]),
    ([(1023,), (4097,), (33, 65)], [F, B, H]),
    ([(3136, 1024), (1024, 10), (10,), (1024,), (5, 5, 32, 64), (64,), (5, 5, 1, 32), (32,)], [F] * 8),
    ([(7,)] * 150 + [(2049,)] * 50, [B, F] * 100),          # many small tensors
    ([(1 << 22,), (3,)], [B, F]),
]


@gpu
@pytest.mark.parametrize("k", range(len(LISTS)))
def test_norm(gpu_lib, k):
    tensors = make(*LISTS[k], seed=k)
    want = float(R.global_norm(tensors))
    plan = GlobalNormClip(tensors)
    got = plan.norm()
    assert got.dtype == torch.float32 and got.shape == ()
    assert abs(float(got) - want) <= want * norm_tol(tensors)
    assert float(plan.norm(scale=0.125)) == float(got) * 0.125      # a power of two moves no bit
    assert torch.equal(plan.norm(), got)                           # bitwise reproducible


@gpu
@pytest.mark.parametrize("k", range(len(LISTS)))
@pytest.mark.parametrize("factor", [0.3, 1.5])
@pytest.mark.parametrize("in_place", [True, False])
def test_clip(gpu_lib, k, factor, in_place):
    tensors = make(*LISTS[k], seed=k + 50)
    before = [t.clone() for t in tensors]
    norm = float(R.global_norm(tensors))
    limit = factor * norm
    out = None if in_place else [torch.full_like(t, 7.0) for t in tensors]
    got, n = GlobalNormClip(tensors, out=out).clip(limit)
    assert abs(float(n) - norm) <= norm * norm_tol(tensors)
    for t, b, o in zip(tensors, before, got):
        if factor > 1.0:
            assert torch.equal(o, b)
        else:
            check_values(o, b.double() * factor_of(norm, limit), b.dtype)
        if not in_place:
            assert torch.equal(t, b)
    if in_place:
        assert all(a is b for a, b in zip(got, tensors))


@gpu
def test_clip_scales_first(gpu_lib):
    tensors = make([(1000,), (77, 3)], [F, B], seed=3)
    norm = float(R.global_norm(tensors, 0.25))
    for limit in (0.5 * norm, 2.0 * norm):
        out, n = GlobalNormClip(tensors, out=[torch.empty_like(t) for t in tensors]).clip(limit, scale=0.25)
        assert abs(float(n) - norm) <= norm * norm_tol(tensors)
        for t, o in zip(tensors, out):
            check_values(o, t.double() * factor_of(norm, limit, 0.25), t.dtype)


@gpu
@pytest.mark.parametrize("dtype", [F, B, H])
def test_strided_and_unaligned_tensors(gpu_lib, dtype):
    """Slices with odd offsets and pitches; what lies between them keeps its values."""
    g = torch.Generator(device=DEV).manual_seed(9)

    def views(buf):
        m = buf[5:5 + 70 * 130].view(70, 130)
        flat = buf[10001:]
        return [m[:, 3:20], m[1:, 40:104], m[:, 129], flat[1:1001], flat[1001:1009].view(2, 4).t(), flat[2000:2000 + 64 * 24].view(64, 24)[:, :16]]

    buf = (torch.randn(20000, device=DEV, generator=g) * 1e-2).to(dtype)
    start = buf.clone()
    tensors = views(buf)
    norm = float(R.global_norm(tensors))
    assert abs(float(GlobalNormClip(tensors).norm()) - norm) <= norm * norm_tol(tensors)
    got, _ = GlobalNormClip(tensors).clip(0.4 * norm)
    for o, b in zip(got, views(start)):
        check_values(o, b.double() * 0.4, dtype)
    touched = torch.zeros_like(buf, dtype=torch.bool)
    for v in views(touched):
        v.fill_(True)
    assert torch.equal(buf[~touched], start[~touched])
    # outputs with another pitch than the tensors
    other = torch.full((70, 50), 3.0, device=DEV).to(dtype)
    src = views(start)[0]
    GlobalNormClip([src], out=[other[:, 1:18]]).clip(1e-3)
    check_values(other[:, 1:18], src.double() * (1e-3 / float(R.global_norm([src]))), dtype)
    assert bool((other[:, 0] == 3).all()) and bool((other[:, 18:] == 3).all())


@gpu
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_a_norm_that_is_not_finite_shows_in_every_value(gpu_lib, bad):
    tensors = make([(5000,), (3,)], [F, B])
    tensors[0][4321] = bad
    out, norm = GlobalNormClip(tensors, out=[torch.zeros_like(t) for t in tensors]).clip(1.0)
    assert not math.isfinite(float(norm))
    assert all(bool(torch.isnan(o).all()) for o in out)
    GlobalNormClip(tensors).clip(1.0)
    assert all(bool(torch.isnan(t).all()) for t in tensors)


@gpu
def test_large_and_small_magnitudes(gpu_lib):
    """Squares of these values leave fp32's range on either side; the norm does not."""
    for scale in (1e30, 1e-30):
        t = make([(4099,)], [F], seed=4, scale=scale)
        norm = float(R.global_norm(t))
        assert abs(float(GlobalNormClip(t).norm()) - norm) <= norm * norm_tol(t)
        want = t[0].double() * 0.5
        GlobalNormClip(t).clip(0.5 * norm)
        check_values(t[0], want, F)


@gpu
def test_elements_beyond_32_bits(gpu_lib):
    n = (1 << 32) + 12345
    t = torch.zeros(n, dtype=B, device=DEV)
    t[5], t[1 << 31], t[n - 1] = 3.0, 4.0, 12.0
    plan = GlobalNormClip([t])
    assert float(plan.norm()) == 13.0
    plan.clip(6.5)
    assert [float(t[k]) for k in (5, 1 << 31, n - 1)] == [1.5, 2.0, 6.0]
    del plan, t
    torch.cuda.empty_cache()


@gpu
def test_the_same_tensor_twice(gpu_lib):
    t = make([(100,)], [F])[0]
    plan = GlobalNormClip([t, t])
    assert float(plan.norm()) == pytest.approx(math.sqrt(2.0) * float(t.double().norm()), rel=1e-6)
    with pytest.raises(ValueError, match="cannot be clipped in place"):
        plan.clip(1.0)
    out = [torch.empty_like(t), torch.empty_like(t)]
    GlobalNormClip([t, t], out=out).clip(1e9)
    assert torch.equal(out[0], t) and torch.equal(out[1], t)


@gpu
def test_refused_limits(gpu_lib):
    plan = GlobalNormClip(make([(10,)], [F]))
    for bad in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(ValueError, match="clip_norm"):
            plan.clip(bad)
    for bad in (-1.0, math.nan, math.inf):
        with pytest.raises(ValueError, match="scale"):
            plan.norm(scale=bad)


def test_table_refuses_bad_spans():
    """dtf_clip_table is host code: no GPU needed."""
    import ctypes
    from distributed_tensorflow_amd.ops import native
    from distributed_tensorflow_amd.ops.clip import ClipSpan
    lib = native.load()
    p = 1 << 20

    def chunks(**kw):
        s = (ClipSpan * 1)(ClipSpan(**{**dict(inp=p, out=p, n=64, in_pitch=0, out_pitch=0, cols=0, dtype=0), **kw}))
        return lib.dtf_clip_table(1, s, None, 0, None)

    assert chunks() == 1 and chunks(n=0, inp=None) == 0 and chunks(n=1025) == 2 and chunks(n=1025, dtype=1) == 1
    assert chunks(n=64, cols=8, in_pitch=9, out_pitch=8) == 1
    for bad in (dict(inp=None), dict(out=None), dict(inp=p + 2), dict(out=p + 2), dict(inp=p + 1, dtype=1), dict(n=-1), dict(dtype=3),
                dict(cols=8, in_pitch=7, out_pitch=8), dict(cols=8, in_pitch=8, out_pitch=7), dict(cols=-1), dict(cols=7, in_pitch=7, out_pitch=7)):
        assert chunks(**bad) == -3, bad
    many = (ClipSpan * 3)(*[ClipSpan(p, p, 5, 0, 0, 0, 0)] * 3)
    room = ctypes.create_string_buffer(128)
    assert lib.dtf_clip_table(3, many, room, 2, None) == -2 and lib.dtf_clip_table(-1, many, None, 0, None) == -3
    assert lib.dtf_clip_partials(5) == 5 and lib.dtf_clip_partials(1 << 20) == 2048 and lib.dtf_clip_partials(-1) == -3


@gpu
def test_native_entries_refuse(gpu_lib):
    t = torch.zeros(64, device=DEV)
    plan = GlobalNormClip([t])
    part = torch.zeros(64, dtype=torch.float64, device=DEV)
    p, q, s = t.data_ptr(), part.data_ptr(), torch.cuda.current_stream().cuda_stream
    table = plan.table.data_ptr()
    assert gpu_lib.dtf_global_norm(None, 1, q, 64, 1.0, None, None, 0, 0.0, p, s) == -3
    assert gpu_lib.dtf_global_norm(table + 8, 1, q, 64, 1.0, None, None, 0, 0.0, p, s) == -3
    assert gpu_lib.dtf_global_norm(table, -1, q, 64, 1.0, None, None, 0, 0.0, p, s) == -3
    assert gpu_lib.dtf_global_norm(table, 1, None, 64, 1.0, None, None, 0, 0.0, p, s) == -3
    assert gpu_lib.dtf_global_norm(table, 1, q, 0, 1.0, None, None, 0, 0.0, p, s) == -3
    assert gpu_lib.dtf_global_norm(table, 1, q, 64, 1.0, None, None, 0, 0.0, None, s) == -3
    assert gpu_lib.dtf_global_norm(table, 1, q, 64, 1.0, p, None, 12, 1.0, None, s) == -3
    assert gpu_lib.dtf_global_norm(table, 1, q, 64, 1.0, p, p, 4, 1.0, None, s) == -3
    assert gpu_lib.dtf_global_norm(table, 1, q, 64, 1.0, p, p, 12, 0.0, None, s) == -3
    assert gpu_lib.dtf_clip_by_global_norm(table, 1, 1, q, 64, 1.0, 0.0, p, s) == -3
    assert gpu_lib.dtf_clip_by_global_norm(table, 1, 1, q, 64, 1.0, math.inf, p, s) == -3
    assert gpu_lib.dtf_clip_by_global_norm(table, 1, 1, q, 64, 1.0, 1.0, None, s) == -3


# ---------------------------------------------------------------------------------------------- streams and graphs
@gpu
def test_graph_replays_follow_the_values(gpu_lib):
    """Two captured graphs over the same tensors, replayed in turn with eager calls between them."""
    tensors = make([(30011,), (513, 7)], [F, B], seed=1)
    outs = [[torch.empty_like(t) for t in tensors] for _ in range(2)]
    plans = [GlobalNormClip(tensors, out=o) for o in outs]
    for p in plans:
        p.clip(0.5)
    torch.cuda.synchronize()
    graphs, norms = [], []
    for p, limit in zip(plans, (0.5, 0.01)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            _, n = p.clip(limit)
        graphs.append(g)
        norms.append(n)
    for rep in range(4):
        for t, fresh in zip(tensors, make([(30011,), (513, 7)], [F, B], seed=100 + rep)):
            t.copy_(fresh)
        eager = float(GlobalNormClip(tensors).norm())
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        norm = float(R.global_norm(tensors))
        for o, n, limit in zip(outs, norms, (0.5, 0.01)):
            assert float(n) == eager
            for t, x in zip(tensors, o):
                check_values(x, t.double() * factor_of(norm, limit), t.dtype)


@gpu
def test_two_streams_at_once(gpu_lib):
    sets = [make([(1 << 20,), (999,)], [F, B], seed=s) for s in range(2)]
    want = [[t.clone() for t in s] for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    plans = [GlobalNormClip(s) for s in sets]
    norms = []
    for st, p in zip(streams, plans):
        with torch.cuda.stream(st):
            norms.append(p.clip(0.1)[1])
    torch.cuda.synchronize()
    for s, w, n in zip(sets, want, norms):
        norm = float(R.global_norm(w))
        assert abs(float(n) - norm) <= norm * norm_tol(w)
        for t, b in zip(s, w):
            check_values(t, b.double() * factor_of(norm, 0.1), b.dtype)
