"""Gated linear recurrence (spk_recurrence, its backward pass and its single
step) against the float64 recurrence, with the error the fp32 arithmetic is
allowed (tests/temporal_ref.py)."""
import pytest
import torch

from spikestack_lite_b200 import ops
from spikestack_lite_b200._lib import EngineError
from tests.temporal_ref import Recurrence, assert_within, stored

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def make(B, L, D, form, dtype, seed=0, spread=6.0):
    g = torch.Generator().manual_seed(seed)
    logit = torch.randn(B, L, D, generator=g) + spread * torch.rand(D, generator=g)
    gate = logit if form == "leaky" else torch.sigmoid(logit) * torch.where(torch.rand(D, generator=g) < 0.2, -1.0, 1.0)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return (r(B, L, D).to(dtype), gate.to(dtype), r(B, D), r(B, L, D).to(dtype), r(B, D))


def check(x, gate, state, gh, glast, form, lengths=None, ref=None):
    """Forward and backward of [B, L, D] inputs (CPU) on the GPU against the float64 recurrence."""
    ref = ref or Recurrence(x, gate, state, form, lengths, gh, glast)
    dx, dgate, dstate = (t.cuda().requires_grad_() for t in (x, gate, state))
    lens = None if lengths is None else lengths.cuda()
    h, last = ops.gated_recurrence(dx, dgate, dstate, form=form, lengths=lens)
    assert h.dtype == x.dtype and last.dtype == torch.float32
    grads = torch.autograd.grad((h, last), (dx, dgate, dstate), (gh.cuda(), glast.cuda()))
    assert_within(h, ref.h, stored(ref.h_err, ref.h, x.dtype), "h")
    assert_within(last, ref.last, ref.last_err, "last")
    assert_within(grads[0], ref.dx, stored(ref.dx_err, ref.dx, x.dtype), "dx")
    assert_within(grads[1], ref.dgate, stored(ref.dgate_err, ref.dgate, x.dtype), "dgate")
    assert_within(grads[2], ref.dstate, ref.dstate_err, "dstate")
    with torch.no_grad():  # the inference call gives the same bits
        h2, last2 = ops.gated_recurrence(dx, dgate, dstate, form=form, lengths=lens)
    assert torch.equal(h, h2) and torch.equal(last, last2)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("form", ["leaky", "gate"])
@pytest.mark.parametrize("shape", [(1, 1, 1), (3, 4, 128), (2, 7, 33), (2, 64, 130), (2, 65, 128), (1, 128, 4),
                                   (5, 200, 36), (1, 1025, 256), (3, 513, 197), (40, 3, 12), (1, 9000, 8),
                                   (70, 150, 36), (33, 200, 130), (129, 67, 128)])
def test_matches_float64(shape, form, dtype):
    check(*make(*shape, form, DT[dtype], seed=sum(shape)), form)


@pytest.mark.parametrize("form", ["leaky", "gate"])
@pytest.mark.parametrize("L", [1, 63, 64, 130, 700])
def test_ragged_lengths(form, L):
    B = 9
    x, gate, state, gh, glast = make(B, L, 40, form, torch.float32, seed=L)
    lengths = torch.tensor([0, 1, L, L // 2, max(L - 1, 0), min(64, L), min(65, L), L + 5, -3], dtype=torch.int32)
    ref = Recurrence(x, gate, state, form, lengths, gh, glast)
    for b in range(B):  # what lies behind a row's end is never read
        n = max(0, min(int(lengths[b]), L))
        for t in (x, gate, gh):
            t[b, n:] = float("nan")
    check(x, gate, state, gh, glast, form, lengths, ref)
    check(x, gate, state, gh, glast, form, lengths.long(), ref)


def test_slow_and_fast_channels_keep_their_accuracy():
    # memories of 10^4 steps beside gates at both ends of the range, large initial states
    B, L, D = 2, 3001, 16
    x, gate, state, gh, glast = make(B, L, D, "leaky", torch.float32, seed=5)
    gate[:, :, 0], gate[:, :, 1], gate[:, :, 2] = 9.5, -9.5, 40.0
    gate[:, :, 3], gate[:, :, 4] = -90.0, 120.0
    state *= 1e3
    check(x, gate, state, gh, glast, "leaky")
    # the gate form beyond 1 and at 0
    x, gate, state, gh, glast = make(B, 200, D, "gate", torch.float32, seed=6)
    gate[:, :, 0], gate[:, :, 1], gate[:, :, 2] = 1.0, 0.0, 1.02
    gate[:, ::7, 3] = 0.0
    check(x, gate, state, gh, glast, "gate")


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_time_planes_and_other_dimensions(dtype):
    # (T, B, N, d) over dim 0, (B, T, N, d) over dim 1, (B, N, T, d) over dim -2
    x, gate, state, gh, glast = make(6, 70, 32, "leaky", DT[dtype], seed=2)
    ref = Recurrence(x, gate, state, "leaky", None, gh, glast)
    base = ops.gated_recurrence(x.cuda(), gate.cuda(), state.cuda())
    assert_within(base[0], ref.h, stored(ref.h_err, ref.h, DT[dtype]), "h")
    for dim in (0, 1, 2):
        view = lambda t: t.view(2, 3, 70, 32).movedim(2, dim).contiguous().cuda()  # noqa: E731
        xs, gs, ghs = view(x).requires_grad_(), view(gate).requires_grad_(), view(gh)
        ss, gl = state.view(2, 3, 32).cuda().requires_grad_(), glast.view(2, 3, 32).cuda()
        h, last = ops.gated_recurrence(xs, gs, ss, dim=dim)
        assert h.shape == xs.shape and last.shape == ss.shape
        assert_within(h.movedim(dim, 2).reshape(6, 70, 32), ref.h, stored(ref.h_err, ref.h, DT[dtype]), f"h dim {dim}")
        dx, dg, ds = torch.autograd.grad((h, last), (xs, gs, ss), (ghs, gl))
        assert_within(dx.movedim(dim, 2).reshape(6, 70, 32), ref.dx, stored(ref.dx_err, ref.dx, DT[dtype]), "dx")
        assert_within(dg.movedim(dim, 2).reshape(6, 70, 32), ref.dgate, stored(ref.dgate_err, ref.dgate, DT[dtype]),
                      "dgate")
        assert_within(ds.reshape(6, 32), ref.dstate, ref.dstate_err, "dstate")


def test_slices_broadcasts_and_misaligned_views():
    x, gate, state, gh, glast = make(3, 90, 34, "leaky", torch.bfloat16, seed=3)
    ref = Recurrence(x, gate, state, "leaky", None, gh, glast)
    both = torch.cat([x, gate], -1).cuda()  # halves of one projection: rows of 68
    h, last = ops.gated_recurrence(both[..., :34], both[..., 34:], state.cuda())
    assert_within(h, ref.h, stored(ref.h_err, ref.h, torch.bfloat16), "slices")
    flat = torch.zeros(x.numel() + 1, dtype=torch.bfloat16, device="cuda")  # one element off any 4-byte boundary
    flat[1:] = x.reshape(-1).cuda()
    h2, last2 = ops.gated_recurrence(flat[1:].view(x.shape), gate.cuda(), state.cuda())
    assert torch.equal(h, h2) and torch.equal(last, last2)
    # every other column is no contiguous last dimension: copied
    wide = torch.repeat_interleave(x, 2, -1).cuda()
    assert torch.equal(ops.gated_recurrence(wide[..., ::2], gate.cuda(), state.cuda())[0], h)
    # one gate for all channels' time steps: a broadcast view, its gradient summed
    lam = torch.randn(34).bfloat16()
    want = Recurrence(x, lam.expand(3, 90, 34), state, "leaky", None, gh, glast)
    lam_d = lam.cuda().requires_grad_()
    h, last = ops.gated_recurrence(x.cuda(), lam_d.expand(3, 90, 34), state.cuda())
    assert_within(h, want.h, stored(want.h_err, want.h, torch.bfloat16), "broadcast gate")
    (dlam,) = torch.autograd.grad((h, last), (lam_d,), (gh.cuda(), glast.cuda()))
    total = want.dgate.sum((0, 1))
    # the elements rounded to bf16, their sum rounded at each of at most 270 additions in fp32 and once to bf16
    err = (want.dgate_err + want.dgate.abs() * 2.0 ** -8 * 1.01 + 270 * 2.0 ** -24 * want.dgate.abs()).sum((0, 1))
    assert_within(dlam, total, stored(err, total, torch.bfloat16), "broadcast gate's gradient")
    # gradients that come broadcast (of a sum) and only for one of the outputs
    xd, gd, sd = x.float().cuda().requires_grad_(), gate.float().cuda().requires_grad_(), state.cuda().requires_grad_()
    ones, zero = torch.ones(3, 90, 34), torch.zeros(3, 34)
    want = Recurrence(x, gate, state, "leaky", None, ones, zero)
    grads = torch.autograd.grad(ops.gated_recurrence(xd, gd, sd)[0].sum(), (xd, gd, sd))
    for got, name in zip(grads, ("dx", "dgate", "dstate")):
        assert_within(got, getattr(want, name), getattr(want, name + "_err"), name)
    want = Recurrence(x, gate, state, "leaky", None, 0 * ones, zero + 1)
    grads = torch.autograd.grad(ops.gated_recurrence(xd, gd, sd)[1].sum(), (xd, gd, sd))
    for got, name in zip(grads, ("dx", "dgate", "dstate")):
        assert_within(got, getattr(want, name), getattr(want, name + "_err"), name)


def test_gradients_against_differences():
    # central differences of the float64 recurrence agree with the kernel's gradients
    x, gate, state, gh, glast = make(1, 6, 3, "leaky", torch.float32, seed=9, spread=0.0)
    xs = [t.cuda().requires_grad_() for t in (x, gate, state)]
    h, last = ops.gated_recurrence(*xs)
    grads = torch.autograd.grad((h, last), xs, (gh.cuda(), glast.cuda()))

    def loss(x, gate, state):
        r = Recurrence(x, gate, state, "leaky")
        return (r.h * gh.double()).sum() + (r.last * glast.double()).sum()

    for k, base in enumerate((x.double(), gate.double(), state.double())):
        for i in range(base.numel()):
            vals = []
            for sign in (1, -1):
                args = [x.double(), gate.double(), state.double()]
                moved = base.clone().view(-1)
                moved[i] += sign * 1e-5
                args[k] = moved.view(base.shape)
                vals.append(loss(*args))
            diff = (vals[0] - vals[1]) / 2e-5
            # the third derivative times 1e-10 / 6 and 1e-16 / 1e-5 of rounding; the kernel's fp32 error
            assert abs(diff - grads[k].double().cpu().reshape(-1)[i]) < 1e-5 * (1 + abs(diff))


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("form", ["leaky", "gate"])
def test_steps_follow_the_recurrence(form, dtype):
    x, gate, state, _, _ = make(5, 9, 37, form, DT[dtype], seed=4)
    ref = Recurrence(x, gate, state, form)
    s = state.cuda()
    for t in range(9):
        out, new = ops.gated_recurrence_step(x[:, t].cuda(), gate[:, t].cuda(), s, form=form)
        assert_within(out, ref.h[:, t], stored(ref.h_err[:, t], ref.h[:, t], DT[dtype]), f"step {t}")
        out2, same = ops.gated_recurrence_step(x[:, t].cuda(), gate[:, t].cuda(), s, form=form, new_state=s)
        assert same is s and torch.equal(out, out2) and torch.equal(s, new)
    assert_within(s, ref.last, ref.last_err, "state")
    # halves of one projection, and every other row of a larger tensor
    both = torch.cat([x[:, 0], gate[:, 0]], -1).cuda()
    want = ops.gated_recurrence_step(x[:, 0].cuda(), gate[:, 0].cuda(), state.cuda(), form=form)
    for xs, gs in ((both[:, :37], both[:, 37:]), (x.cuda()[:, 0], gate.cuda()[:, 0])):
        got = ops.gated_recurrence_step(xs, gs, state.cuda(), form=form)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # split in two calls through the state
    a = ops.gated_recurrence(x[:, :4].cuda(), gate[:, :4].cuda(), state.cuda(), form=form)
    b = ops.gated_recurrence(x[:, 4:].cuda(), gate[:, 4:].cuda(), a[1], form=form)
    assert_within(torch.cat([a[0], b[0]], 1), ref.h, stored(ref.h_err, ref.h, DT[dtype]), "two calls")


def test_empty_and_non_finite():
    dev = "cuda"
    s = torch.randn(2, 5, device=dev, requires_grad=True)
    x = torch.empty(2, 0, 5, device=dev, requires_grad=True)
    h, last = ops.gated_recurrence(x, torch.empty(2, 0, 5, device=dev), s)
    assert h.shape == (2, 0, 5) and torch.equal(last, s)
    (gs,) = torch.autograd.grad(last, s, torch.ones_like(last))
    assert torch.equal(gs, torch.ones_like(gs))
    h, last = ops.gated_recurrence(torch.empty(0, 4, 5, device=dev), torch.empty(0, 4, 5, device=dev))
    assert h.shape == (0, 4, 5) and last.shape == (0, 5)
    # a NaN or an infinity spoils its own channel from its step on, and no other
    x, gate, state, _, _ = make(1, 300, 8, "leaky", torch.float32, seed=8)
    clean = ops.gated_recurrence(x.cuda(), gate.cuda(), state.cuda())[0]
    x[0, 100, 2], x[0, 150, 5] = float("nan"), float("inf")
    h = ops.gated_recurrence(x.cuda(), gate.cuda(), state.cuda())[0]
    keep = [0, 1, 3, 4, 6, 7]
    assert torch.equal(h[..., keep], clean[..., keep])
    assert torch.equal(h[:, :100], clean[:, :100])
    assert not h[0, 100:, 2].isfinite().any() and not h[0, 150:, 5].isfinite().any()


@pytest.mark.parametrize("form", ["leaky", "gate"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("L", [3, 40, 300])
def test_non_finite_gates(L, dtype, form):
    x, gate, state, _, _ = make(2, L, 8, form, DT[dtype], seed=L)
    clean = ops.gated_recurrence(x.cuda(), gate.cuda(), state.cuda(), form=form)[0]
    gate[0, L // 2, 2] = float("nan")
    h, last = ops.gated_recurrence(x.cuda(), gate.cuda(), state.cuda(), form=form)
    assert h[0, L // 2:, 2].isnan().all() and last[0, 2].isnan()
    h[0, L // 2:, 2] = clean[0, L // 2:, 2]
    assert torch.equal(h, clean)
    if form == "leaky":  # gates without bound: the input itself, or the state kept
        gate[0, L // 2, 2], gate[1, 0, 3] = -float("inf"), float("inf")
        h, _ = ops.gated_recurrence(x.cuda(), gate.cuda(), state.cuda())
        assert h.isfinite().all()
        assert h[0, L // 2, 2] == x[0, L // 2, 2] and h[1, 0, 3] == state[1, 3].to(DT[dtype])


def test_lengths_of_planes_and_one_sided_gradients():
    # (T, B, N, d) over dim 0 with a length per (b, n); gradients of x alone, of the gate alone
    x, gate, state, gh, glast = make(6, 33, 20, "leaky", torch.float32, seed=11)
    lengths = torch.tensor([0, 33, 5, 1, 32, 17])
    ref = Recurrence(x, gate, state, "leaky", lengths, gh, glast)
    view = lambda t: t.view(2, 3, 33, 20).movedim(2, 0).contiguous().cuda()  # noqa: E731
    back = lambda t: t.movedim(0, 2).reshape(6, 33, 20)  # noqa: E731
    xs, gs, ss = view(x), view(gate), state.view(2, 3, 20).cuda()
    for mine, want, err in ((xs, ref.dx, ref.dx_err), (gs, ref.dgate, ref.dgate_err)):
        mine.requires_grad_()
        h, last = ops.gated_recurrence(xs, gs, ss, dim=0, lengths=lengths.view(2, 3).cuda())
        assert_within(back(h), ref.h, stored(ref.h_err, ref.h, torch.float32), "h")
        (got,) = torch.autograd.grad((h, last), mine, (view(gh), glast.view(2, 3, 20).cuda()))
        assert_within(back(got), want, stored(err, want, torch.float32), "gradient")
        mine.requires_grad_(False)
    # x as its own gate: both gradients arrive
    x.requires_grad_(False)
    both = x.cuda().requires_grad_()
    h, last = ops.gated_recurrence(both, both, state.cuda())
    (got,) = torch.autograd.grad((h, last), both, (gh.cuda(), glast.cuda()))
    own = Recurrence(x, x, state, "leaky", None, gh, glast)
    assert_within(got, own.dx + own.dgate, own.dx_err + own.dgate_err + 2.0 ** -23 * (own.dx.abs() + own.dgate.abs()),
                  "x as its own gate")


def test_no_second_derivative():
    x = torch.randn(2, 5, 8, device="cuda", requires_grad=True)
    h, _ = ops.gated_recurrence(x, x)
    (g,) = torch.autograd.grad(h.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_offsets_beyond_32_bits():
    # 2.3e9 elements: the inputs broadcast along time, the states written out; constant gates have a closed form
    L, D = 70000, 33000
    g = torch.Generator().manual_seed(12)
    x, gate, state = (torch.randn(1, D, generator=g) for _ in range(3))
    gate = (gate + 6).bfloat16()
    x = x.bfloat16()
    h, last = ops.gated_recurrence(x.cuda().expand(1, L, D), gate.cuda().expand(1, L, D), state.cuda())
    a = torch.sigmoid(gate.double())
    for t in (0, 1000, 65535, L - 1):
        want = a ** (t + 1) * state.double() + (1 - a ** (t + 1)) * x.double()
        # a memory of 1 / (1 - a) steps, each off by a few u of the state: (see Recurrence)
        err = 40 * 2.0 ** -24 * (1 / (1 - a)).clamp(max=t + 1) * (state.abs() + x.abs()).double()
        assert_within(h[:, t], want, stored(err, want, torch.bfloat16), f"step {t}")
    assert_within(last, want, err, "last")


def test_runs_on_a_side_stream_and_in_a_graph():
    x, gate, state, gh, glast = make(2, 300, 64, "leaky", torch.float32, seed=1)
    x, gate, state, gh, glast = (t.cuda() for t in (x, gate, state, gh, glast))

    def train(x, gate, state):
        x, gate, state = (t.detach().requires_grad_() for t in (x, gate, state))
        h, last = ops.gated_recurrence(x, gate, state)
        return (h.detach(), last.detach(), *torch.autograd.grad((h, last), (x, gate, state), (gh, glast)))

    want = train(x, gate, state)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = train(x, gate, state)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    bufs = [torch.zeros_like(t) for t in (x, gate, state)]
    graphs = []
    for _ in range(2):  # two captured graphs share nothing but their inputs
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = train(*bufs)
        graphs.append((graph, out))
    for b, t in zip(bufs, (x, gate, state)):
        b.copy_(t)
    streams = [torch.cuda.Stream() for _ in graphs]
    for (graph, _), st in zip(graphs, streams):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            for _ in range(3):
                graph.replay()
    for st in streams:
        torch.cuda.current_stream().wait_stream(st)
    for _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(want, out))


def test_refusals():
    x = torch.randn(2, 4, 8, device="cuda")
    s = torch.zeros(2, 8, device="cuda")
    for bad in (dict(gate=x[:, :3]), dict(gate=x.half()), dict(form="tanh"), dict(form=None), dict(dim=-1),
                dict(dim=2), dict(dim=5), dict(state=s[:1]), dict(state=s.half()), dict(lengths=torch.zeros(2, device="cuda")),
                dict(lengths=torch.zeros(3, dtype=torch.int32, device="cuda")), dict(state=s.cpu()),
                dict(x=x.double(), gate=x.double())):
        args = dict(x=x, gate=x)
        args.update(bad)
        with pytest.raises(EngineError):
            ops.gated_recurrence(**args)
    for bad in (dict(gate=x[0, 1:]), dict(state=x[0].half()), dict(form=1), dict(new_state=x[0].half()),
                dict(new_state=torch.zeros(8, 4, device="cuda").t()), dict(x=x[0].detach().requires_grad_())):
        args = dict(x=x[0], gate=x[0], state=x[0])
        args.update(bad)
        with pytest.raises(EngineError):
            ops.gated_recurrence_step(**args)
