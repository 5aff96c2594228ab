"""Group norm with an activation, channels last (spk_group_norm_act and its
backward pass), against the float64 formulas with the error the fp32
arithmetic is allowed (tests/temporal_ref.py)."""
import pytest
import torch

from spikestack_lite_b200 import ops
from spikestack_lite_b200._lib import EngineError
from tests.temporal_ref import GroupNorm, assert_within, stored

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SHAPES = [(1, 1, 1, 1), (3, 64, 128, 8), (2, 1, 32, 8), (5, 7, 33, 11), (2, 301, 330, 10), (1, 1000, 12, 3),
          (7, 13, 96, 1), (2, 130, 64, 64), (3, 50, 520, 4), (1, 5000, 40, 5), (300, 3, 16, 2), (1, 40, 4112, 16), (2, 3, 6000, 3000), (1, 5, 24576, 24576),
          (2, 2500, 256, 32)]


def make(S, P, C, dtype, seed=0, shift=0.5):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x = (r(S, P, C) * (0.5 + torch.rand(C, generator=g)) + shift).to(dtype)
    return x, 1 + 0.2 * r(C), 0.2 * r(C), r(S, P, C).to(dtype)


def check(x, groups, w, b, gy, act, eps=1e-5, thr=0.0):
    ref = GroupNorm(x, groups, w, b, eps, act, thr, gy)
    xd = x.cuda().requires_grad_()
    wd = None if w is None else w.cuda().requires_grad_()
    bd = None if b is None else b.cuda().requires_grad_()
    y = ops.group_norm_act(xd, groups, wd, bd, eps=eps, act=act, thr=thr)
    assert y.dtype == x.dtype
    ins = [t for t in (xd, wd, bd) if t is not None]
    grads = list(torch.autograd.grad(y, ins, gy.cuda()))
    assert_within(y, ref.y, stored(ref.y_err, ref.y, x.dtype), "y")
    assert_within(grads.pop(0), ref.dx, stored(ref.dx_err, ref.dx, x.dtype), "dx")
    if w is not None:
        assert_within(grads.pop(0), ref.dweight, ref.dweight_err, "dweight")
    if b is not None:
        assert_within(grads.pop(0), ref.dbias, ref.dbias_err, "dbias")
    with torch.no_grad():
        assert torch.equal(y, ops.group_norm_act(xd, groups, wd, bd, eps=eps, act=act, thr=thr))


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("act", ["none", "silu", "heaviside"])
@pytest.mark.parametrize("shape", SHAPES)
def test_matches_float64(shape, act, dtype):
    S, P, C, G = shape
    x, w, b, gy = make(S, P, C, DT[dtype], seed=S + P + C)
    check(x, G, w, b, gy, act, thr=0.25)


def test_spikes_away_from_the_threshold_are_exact():
    x, w, b, gy = make(4, 256, 64, torch.float32, seed=1)
    ref = GroupNorm(x, 8, w, b, 1e-5, "heaviside", 0.1)
    y = ops.group_norm_act(x.cuda(), 8, w.cuda(), b.cuda(), act="heaviside", thr=0.1).double().cpu()
    assert set(y.unique().tolist()) <= {0.0, 1.0}
    assert (ref.y_err > 0).double().mean() < 1e-3  # the band in which rounding decides is thin
    assert torch.equal(y[ref.y_err == 0], ref.y[ref.y_err == 0])


def test_no_affine_parameters_and_one_of_them():
    x, w, b, gy = make(3, 70, 48, torch.float32, seed=2)
    check(x, 6, None, None, gy, "silu")
    check(x, 6, w, None, gy, "silu")
    check(x, 6, None, b, gy, "silu")


def test_large_means_outliers_and_constant_groups():
    # a mean far above the spread: no difference of large sums
    x, w, b, gy = make(2, 300, 64, torch.float32, seed=3, shift=3000.0)
    check(x, 8, w, b, gy, "none")
    # the first element of a group far from all the others
    x, w, b, gy = make(2, 300, 64, torch.float32, seed=4)
    x[:, 0, ::8] = 1e4
    check(x, 8, w, b, gy, "silu")
    # constant groups: x - mean is rounding, y = act(bias) to its size
    x = torch.full((2, 40, 16), 0.75)
    y = ops.group_norm_act(x.cuda(), 4, None, torch.arange(16.0).cuda())
    assert torch.equal(y.cpu(), torch.arange(16.0).expand(2, 40, 16))
    # values whose square leaves fp16's range: the statistics are fp32
    x, w, b, gy = make(2, 64, 32, torch.float16, seed=5)
    check(x * 1000, 4, w, b, gy, "none")


def test_leading_dimensions_and_views():
    x, w, b, gy = make(6, 35, 24, torch.bfloat16, seed=6)
    want = ops.group_norm_act(x.cuda(), 3, w.cuda(), b.cuda(), act="silu")
    assert torch.equal(ops.group_norm_act(x.view(6, 5, 7, 24).cuda(), 3, w.cuda(), b.cuda(), act="silu").view_as(want),
                       want)
    wide = torch.cat([x, x], -1).cuda()
    assert torch.equal(ops.group_norm_act(wide[..., 24:], 3, w.cuda(), b.cuda(), act="silu"), want)
    flat = torch.zeros(x.numel() + 1, dtype=torch.bfloat16, device="cuda")  # one element off its alignment
    flat[1:] = x.reshape(-1).cuda()
    got = ops.group_norm_act(flat[1:].view(x.shape), 3, w.cuda(), b.cuda(), act="silu")
    ref = GroupNorm(x, 3, w, b, 1e-5, "silu")
    assert_within(got, ref.y, stored(ref.y_err, ref.y, torch.bfloat16), "misaligned")
    two = ops.group_norm_act(x[:, 0].cuda(), 3)  # (samples, channels): one position
    ref = GroupNorm(x[:, :1], 3, None, None, 1e-5, "none")
    assert_within(two.unsqueeze(1), ref.y, stored(ref.y_err, ref.y, torch.bfloat16), "one position")


def test_empty_inputs():
    w = torch.ones(8, device="cuda", requires_grad=True)
    for shape in ((0, 5, 8), (3, 0, 8)):
        x = torch.empty(*shape, device="cuda", requires_grad=True)
        y = ops.group_norm_act(x, 2, w)
        assert y.shape == shape
        gx, gw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
        assert gx.shape == shape and torch.equal(gw, torch.zeros_like(gw))


def test_non_finite_values_stay_in_their_group():
    x, w, b, gy = make(3, 64, 32, torch.float32, seed=7)
    want = ops.group_norm_act(x.cuda(), 4, w.cuda(), b.cuda())
    x[1, 5, 9] = float("inf")
    x[2, 6, 30] = float("nan")
    y = ops.group_norm_act(x.cuda(), 4, w.cuda(), b.cuda())
    touched = torch.zeros_like(x, dtype=torch.bool)
    touched[1, :, 8:16] = True
    touched[2, :, 24:32] = True
    assert torch.equal(y[~touched.cuda()], want[~touched.cuda()])
    assert y[touched.cuda()].isnan().any()


def test_parameter_gradients_are_the_same_bits_every_run():
    x, w, b, gy = make(64, 200, 128, torch.bfloat16, seed=8)
    runs = []
    for _ in range(4):
        xd, wd, bd = x.cuda().requires_grad_(), w.cuda().requires_grad_(), b.cuda().requires_grad_()
        y = ops.group_norm_act(xd, 8, wd, bd, act="silu")
        runs.append((y.detach(), *torch.autograd.grad(y, (xd, wd, bd), gy.cuda())))
    for r in runs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(r, runs[0]))


@pytest.mark.parametrize("shape", [(300, 300, 64, 4), (2, 900, 256, 8), (3, 1500, 96, 2), (40, 700, 40, 4)])
def test_samples_in_clusters_and_in_tiles(shape):
    # sizes at which the blocks of a cluster share a sample, forward, backward or both
    S, P, C, G = shape
    for dtype in (torch.float32, torch.bfloat16):
        x, w, b, gy = make(S, P, C, dtype, seed=P)
        check(x, G, w, b, gy, "silu")


def test_offsets_beyond_32_bits():
    # 2.3e9 elements: one row pattern repeated, whose group statistics are those of the row
    P, C, G = 70000, 33024, 4
    row = torch.randn(C, generator=torch.Generator().manual_seed(3)).bfloat16()
    x = row.cuda().expand(1, P, C).contiguous()
    y = ops.group_norm_act(x, G)
    ref = GroupNorm(row.view(1, 1, C), G, None, None, 1e-5, "none")
    # the mean of P equal rows: their sums take log2(P) + 128 roundings more
    for t in (0, 65535, P - 1):
        assert_within(y[:, t:t + 1], ref.y, stored(2 * ref.y_err, ref.y, torch.bfloat16), f"row {t}")


def test_no_second_derivative():
    x = torch.randn(2, 5, 8, device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad(ops.group_norm_act(x, 2, act="silu").sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.parametrize("shape", [(3, 64, 128, 8), (2, 3000, 512, 32)])
def test_runs_on_a_side_stream_and_in_a_graph(shape):
    S, P, C, G = shape
    x, w, b, gy = (t.cuda() for t in make(S, P, C, torch.float32, seed=9))

    def train(x, w, b):
        x, w, b = (t.detach().requires_grad_() for t in (x, w, b))
        y = ops.group_norm_act(x, G, w, b, act="silu")
        return (y.detach(), *torch.autograd.grad(y, (x, w, b), gy))

    want = train(x, w, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = train(x, w, b)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    bufs = [torch.zeros_like(t) for t in (x, w, b)]
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = train(*bufs)
        graphs.append((graph, out))
    for buf, t in zip(bufs, (x, w, b)):
        buf.copy_(t)
    streams = [torch.cuda.Stream() for _ in graphs]
    for (graph, _), st in zip(graphs, streams):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            for _ in range(3):
                graph.replay()
    for st in streams:
        torch.cuda.current_stream().wait_stream(st)
    for _, out in graphs:
        assert all(torch.equal(p, q) for p, q in zip(want, out))


def test_refusals():
    x = torch.randn(2, 4, 12, device="cuda")
    w = torch.ones(12, device="cuda")
    for args, kw in (((x, 5), {}), ((x, 0), {}), ((x.double(), 3), {}), ((x, 3, w[:6]), {}), ((x, 3, w.half()), {}),
                     ((x, 3, w.cpu()), {}), ((x, 3), {"act": "relu"}), ((x, 3), {"eps": -1.0}), ((x.cpu(), 3), {}),
                     ((x[0, 0], 3), {})):
        with pytest.raises(EngineError):
            ops.group_norm_act(*args, **kw)
