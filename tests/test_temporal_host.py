"""The training and streaming operators without a GPU: argument checks at the
C entry points, the no-CPU-path contract, and the tests' own plain
implementations (Philox against its published known answers, gradients against
central differences)."""
import ctypes

import pytest
import torch

from tests.temporal_ref import GroupNorm, Recurrence, philox


@pytest.fixture(scope="module")
def lib():
    from spikestack_lite_b200 import _lib, build

    build.build()
    return _lib.load()


P = ctypes.c_void_p(256)
ODD = ctypes.c_void_p(257)


def test_philox_known_answers():
    ones = 0xFFFFFFFF
    assert philox((0,) * 4, (0, 0)) == [0x5F6FB709, 0x0D893F64, 0x4F121F81, 0x4F730A48]
    assert philox((ones,) * 4, (ones, ones)) == [0x5207DDC2, 0x45165E59, 0x4D8EE751, 0x8C52F662]
    assert philox((0,) * 4, (0, 0), rounds=10) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]


@pytest.mark.parametrize("form", ["leaky", "gate"])
def test_plain_recurrence_gradients_against_differences(form):
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g).double()  # noqa: E731
    args, gh, gl = [r(3, 5, 2), r(3, 5, 2), r(3, 2)], r(3, 5, 2), r(3, 2)
    lens = torch.tensor([5, 0, 3])
    ref = Recurrence(*args, form, lens, gh, gl)

    def loss(a):
        o = Recurrence(*a, form, lens)
        return (o.h * gh).sum() + (o.last * gl).sum()

    for k, name in enumerate(("dx", "dgate", "dstate")):
        want = getattr(ref, name).reshape(-1)
        for i in range(want.numel()):
            vals = []
            for sign in (1, -1):
                a = [t.clone() for t in args]
                a[k].view(-1)[i] += sign * 1e-5
                vals.append(loss(a))
            # truncation 1e-10 times the third derivative, rounding 1e-15 / 1e-5
            assert abs((vals[0] - vals[1]) / 2e-5 - want[i]) < 1e-7


@pytest.mark.parametrize("act", ["none", "silu"])
def test_plain_group_norm_gradients_against_differences(act):
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g).double()  # noqa: E731
    args, gy = [r(2, 5, 6), r(6), r(6)], r(2, 5, 6)
    ref = GroupNorm(args[0], 2, args[1], args[2], 1e-5, act, 0.0, gy)
    for k, name in enumerate(("dx", "dweight", "dbias")):
        want = getattr(ref, name).reshape(-1)
        for i in range(want.numel()):
            vals = []
            for sign in (1, -1):
                a = [t.clone() for t in args]
                a[k].view(-1)[i] += sign * 1e-5
                vals.append((GroupNorm(a[0], 2, a[1], a[2], 1e-5, act).y * gy).sum())
            assert abs((vals[0] - vals[1]) / 2e-5 - want[i]) < 1e-7


def test_recurrence_entry_points_reject_bad_arguments(lib):
    from spikestack_lite_b200._lib import SPK_EINVAL, SPK_OK

    def fwd(x=P, gate=P, dtype=0, form=1, B=2, L=4, D=8, state=None, lengths=None, h=P, last=P, carry=None):
        return lib.spk_recurrence(x, 32, 8, gate, 32, 8, dtype, form, B, L, D, state, lengths, h, 32, 8, last, carry,
                                  None)

    assert fwd(B=0) == SPK_OK and fwd(D=0) == SPK_OK  # nothing to do
    for bad in (dict(dtype=3), dict(dtype=-1), dict(form=2), dict(B=-1), dict(L=-1), dict(D=-1), dict(x=None),
                dict(gate=None), dict(h=None), dict(last=None), dict(x=ODD), dict(dtype=1, gate=ODD), dict(last=ODD),
                dict(lengths=ODD), dict(state=ODD), dict(L=1 << 31), dict(B=1 << 40, D=1 << 20)):
        assert fwd(**bad) == SPK_EINVAL, bad
        assert lib.spk_last_error()

    def bwd(x=P, gate=P, gh=None, dtype=0, form=1, B=2, L=4, D=8, carry=None, dx=P, dgate=P, glast=None):
        return lib.spk_recurrence_backward(x, 32, 8, gate, 32, 8, gh, 32, 8, dtype, form, B, L, D, None, None, carry,
                                           glast, dx, dgate, 32, 8, None, None)

    assert bwd(B=0) == SPK_OK
    for bad in (dict(dtype=3), dict(form=-1), dict(dx=None), dict(dgate=None), dict(x=None), dict(gh=ODD),
                dict(glast=ODD), dict(L=lib.spk_recurrence_chunk(0, 2, 1 << 20, 8) + 1)):
        assert bwd(**bad) == SPK_EINVAL, bad
    assert b"carry" in lib.spk_last_error()

    def step(x=P, gate=P, dtype=0, form=1, rows=4, D=8, state=P, out=P, new=P):
        return lib.spk_recurrence_step(x, 8, gate, 8, dtype, form, rows, D, state, out, new, None)

    assert step(rows=0) == SPK_OK and step(D=0) == SPK_OK
    for bad in (dict(rows=-1), dict(D=-1), dict(x=None), dict(state=None), dict(out=None), dict(new=None),
                dict(dtype=9), dict(form=7), dict(new=ODD), dict(rows=1 << 40, D=1 << 20)):
        assert step(**bad) == SPK_EINVAL, bad


def test_group_norm_entry_points_reject_bad_arguments(lib):
    from spikestack_lite_b200._lib import SPK_EINVAL, SPK_EWORKSPACE, SPK_OK

    need = lib.spk_group_norm_workspace_bytes(0, 2, 64, 32, 4)
    assert need > 0 and lib.spk_group_norm_workspace_bytes(0, 0, 64, 32, 4) == 0

    def fwd(X=P, dtype=0, S=2, Pn=64, C=32, G=4, w=None, b=None, eps=1e-5, act=0, Y=P, mean=None, rstd=None, ws=P,
            n=need):
        return lib.spk_group_norm_act(X, dtype, S, Pn, C, G, w, b, eps, act, 0.0, Y, mean, rstd, ws, n, None)

    assert fwd(S=0, X=None, Y=None, ws=None, n=0) == SPK_OK
    for bad in (dict(dtype=3), dict(C=0), dict(G=0), dict(G=5), dict(S=-1), dict(Pn=-1), dict(eps=-1.0), dict(act=2),
                dict(act=3), dict(act=9), dict(X=None), dict(Y=None), dict(mean=P), dict(X=ODD), dict(w=ODD),
                dict(ws=ODD), dict(S=1 << 31), dict(C=1 << 21, G=1)):
        assert fwd(**bad) == SPK_EINVAL, bad
    assert fwd(ws=None) == SPK_EWORKSPACE and fwd(n=need - 1) == SPK_EWORKSPACE

    def bwd(X=P, GY=P, mean=P, rstd=P, DX=P, ws=P, n=need, act=0):
        return lib.spk_group_norm_act_backward(X, GY, 0, 2, 64, 32, 4, None, None, mean, rstd, act, 0.0, DX, None,
                                               None, ws, n, None)

    for bad in (dict(X=None), dict(GY=None), dict(mean=None), dict(rstd=None), dict(DX=None), dict(act=4),
                dict(GY=ODD)):
        assert bwd(**bad) == SPK_EINVAL, bad
    assert bwd(ws=None) == SPK_EWORKSPACE


def test_dropout_entry_point_rejects_bad_arguments(lib):
    from spikestack_lite_b200._lib import SPK_EINVAL, SPK_OK

    def call(X=P, R=None, dtype=0, n=8, p=0.5, key=None, Y=P):
        return lib.spk_dropout(X, R, dtype, n, p, 1, 2, key, Y, None)

    assert call(n=0, X=None, Y=None) == SPK_OK
    for bad in (dict(n=-1), dict(p=-0.1), dict(p=1.5), dict(p=float("nan")), dict(dtype=3), dict(X=None),
                dict(Y=None), dict(X=ODD), dict(R=ODD), dict(key=ODD)):
        assert call(**bad) == SPK_EINVAL, bad


def test_python_ops_refuse_cpu_tensors(lib):
    from spikestack_lite_b200 import ops
    from spikestack_lite_b200._lib import EngineError

    x = torch.zeros(2, 4, 8)
    with pytest.raises(EngineError, match="CUDA"):
        ops.gated_recurrence(x, x)
    with pytest.raises(EngineError, match="CUDA"):
        ops.gated_recurrence_step(x, x, x)
    with pytest.raises(EngineError, match="CUDA"):
        ops.group_norm_act(x, 2)
    with pytest.raises(EngineError, match="CUDA"):
        ops.dropout(x, 0.5, (0, 0))


def test_time_strides():
    from spikestack_lite_b200.ops import _empty_time, _time_major, _time_strides

    x = torch.zeros(4, 3, 5, 8)  # (T, B, N, d)
    assert _time_strides(x, 0) == (8, 120)
    assert _time_strides(x, 1) is None  # the planes do not flatten with the tokens around dimension 1
    assert _time_strides(x, 2) == (40, 8)
    assert _time_strides(x.transpose(2, 3), 0) is None
    assert _time_strides(x[:, :, :1], 1) == (120, 40)
    assert _time_strides(x[:, 0], 0) == (8, 120)
    assert _time_strides(x[0, 0, 0].expand(3, 5, 8), 1) == (0, 0)
    t, st = _time_major(x, 1)
    assert t.shape == x.shape and st == _time_strides(t, 1) == (32 * 3 // 4, 8)
    for shape in ((4, 3, 5, 8), (2, 70, 3, 32), (3, 1, 5, 8), (2, 3, 4, 5, 6), (7, 9, 2), (4, 2)):
        for dim in range(len(shape) - 1):  # an output holds exactly the elements that its strides reach
            x = torch.zeros(shape)
            out, (step_b, step_t) = _empty_time(x, dim)
            steps, width = shape[dim], shape[-1]
            rows = x.numel() // (steps * width)
            assert out.shape == x.shape and step_t >= width and (step_b >= width or rows == 1)
            reach = (rows - 1) * step_b + (steps - 1) * step_t + width
            assert reach == x.numel() == out.untyped_storage().nbytes() // 4
            at = torch.arange(rows).view(-1, 1, 1) * step_b + torch.arange(steps).view(-1, 1) * step_t + torch.arange(width)
            out.copy_(torch.arange(x.numel()).view(shape))
            flat = torch.empty(x.numel()).set_(out.untyped_storage())
            want = torch.arange(x.numel()).view(shape).movedim(dim, -2).reshape(rows, steps, width)
            assert torch.equal(flat[at.reshape(-1)].long(), want.reshape(-1))


def test_modules_on_the_host():
    from spikestack_lite_b200._lib import EngineError
    from spikestack_lite_b200.recurrence import Dropout, GatedRecurrence
    from spikestack_lite_b200.transformer import SpikingTransformer

    cfg = dict(temporal=True, n_repeats=3, use_spikeskip=True, expansion=4)
    torch.manual_seed(0)
    plain = SpikingTransformer(**cfg).state_dict()
    torch.manual_seed(0)
    more = SpikingTransformer(**cfg, use_recurrence=True).state_dict()
    assert all(torch.equal(more[k], v) for k, v in plain.items())  # a seed's weights do not change
    assert {k.split(".")[0] for k in set(more) - set(plain)} == {"recurrence"}
    assert set(SpikingTransformer(**cfg, dropout=0.1).state_dict()) == set(plain)  # no mask, no key
    with pytest.raises(ValueError):
        SpikingTransformer(use_recurrence=True)
    with pytest.raises(ValueError):
        GatedRecurrence(10, groups=4)
    with pytest.raises(ValueError):
        Dropout(1.5)
    m = GatedRecurrence(16, groups=4)
    with pytest.raises(EngineError, match="CUDA"):
        m(torch.zeros(3, 2, 5, 16))
    with pytest.raises(EngineError, match="CUDA"):
        m.step(torch.zeros(2, 5, 16))
    d = Dropout(0.5)
    d.manual_seed(7, 3)
    assert d.key.tolist() == [7, 3]
    d.eval()
    x = torch.randn(4)
    assert d(x) is x and torch.equal(d(x, residual=x), x + x) and d.key.tolist() == [7, 3]
