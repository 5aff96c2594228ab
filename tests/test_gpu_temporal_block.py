"""The training and streaming operators together: the GatedRecurrence block
(group norm + SiLU, projection halves, recurrence over the planes, dropout with
the residual), its streaming form, and the model's dropout."""
import pytest
import torch

from spikestack_lite_b200 import ops
from spikestack_lite_b200._lib import EngineError
from spikestack_lite_b200.attention import AstrocyteHebbianBlock
from spikestack_lite_b200.graphs import CapturedForward
from spikestack_lite_b200.recurrence import Dropout, GatedRecurrence
from spikestack_lite_b200.transformer import SpikingTransformer

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def plain_block(m, x, state, keep=None, p=0.0):
    """GatedRecurrence.forward from its formulas in float64 (differentiable)."""
    P = {k: v.detach().double().cpu().requires_grad_() for k, v in m.named_parameters()}
    T, B, N, d = x.shape
    xg = x.reshape(T * B, N, m.groups, d // m.groups)
    var, mean = torch.var_mean(xg, dim=(1, 3), correction=0, keepdim=True)
    z = ((xg - mean) / torch.sqrt(var + m.eps)).reshape(T, B, N, d) * P["norm_weight"] + P["norm_bias"]
    u = z * torch.sigmoid(z)
    vg = u @ P["vg_proj.weight"].t() + P["vg_proj.bias"]
    v, a = vg[..., :d], torch.sigmoid(vg[..., d:])
    h, hs = state, []
    for t in range(T):
        h = a[t] * h + (1 - a[t]) * v[t]
        hs.append(h)
    y = torch.stack(hs) @ P["o_proj.weight"].t() + P["o_proj.bias"]
    if keep is not None:
        y = y * keep / (1 - p)
    return x + y, h, P


def close(got, want, terms, what):
    """Within `terms` roundings of u of the largest value: every result here is a
    chain of sums whose magnitudes stay within ten times the largest result."""
    got, want = got.detach().double().cpu(), want.detach().double()
    err = (got - want).abs().max().item() / want.abs().max().item()
    assert err < 10 * terms * U, f"{what}: {err:.3g}"


@pytest.mark.parametrize("T", [1, 5, 70])
@pytest.mark.parametrize("dropout", [0.0, 0.25])
def test_block_trains(T, dropout):
    torch.manual_seed(T)
    # 64 products per sum, twice; the group statistics (128), T steps of the recurrence at most
    terms = 2 * 64 + 128 + min(T, 64)
    m = GatedRecurrence(64, groups=4, dropout=dropout).cuda()
    x = torch.randn(T, 2, 9, 64, device="cuda", requires_grad=True)
    s0 = torch.randn(2, 9, 64, device="cuda", requires_grad=True)
    gy, gs = torch.randn(T, 2, 9, 64, device="cuda"), torch.randn(2, 9, 64, device="cuda")
    keep = None
    if dropout:
        m.dropout.manual_seed(5, 8)
        keep = (ops.dropout(torch.ones_like(gy), dropout, (5, 8)) != 0).double().cpu()
    y, s = m(x, s0)
    if dropout:
        assert m.dropout.key.tolist() == [5, 9]
    xr, sr = x.detach().double().cpu().requires_grad_(), s0.detach().double().cpu().requires_grad_()
    yr, hr, P = plain_block(m, xr, sr, keep, dropout)
    close(y, yr, terms, "y")
    close(s, hr, terms, "state")
    params = dict(m.named_parameters())
    got = torch.autograd.grad((y, s), [x, s0, *params.values()], (gy, gs))
    want = torch.autograd.grad((yr, hr), [xr, sr, *(P[k] for k in params)], (gy.double().cpu(), gs.double().cpu()))
    # the parameters' gradients add up T * 18 rows more
    for g, w, name in zip(got, want, ["x", "state", *params]):
        close(g, w, 2 * terms + T * 18, name)


def test_a_stream_follows_the_planes():
    torch.manual_seed(1)
    m = GatedRecurrence(128, groups=8, dropout=0.5).cuda().eval()
    x = torch.randn(12, 3, 20, 128, device="cuda")
    with torch.no_grad():
        want, last = m(x)
    state, outs = None, []
    for t in range(12):
        y, state = m.step(x[t], state)
        outs.append(y)
    # the projections run at two batch sizes; each plane's own arithmetic is the same
    terms = 2 * 128 + 128 + 12
    close(torch.stack(outs), want.cpu(), terms, "stream")
    close(state, last.cpu(), terms, "state")
    with torch.no_grad():  # in two parts
        a, s = m(x[:7])
        b, s = m(x[7:], s)
    close(torch.cat([a, b]), want.cpu(), terms, "two parts")


def test_training_step_in_a_graph_draws_new_masks():
    torch.manual_seed(2)
    m = GatedRecurrence(64, groups=4, dropout=0.5).cuda()
    x = torch.randn(4, 2, 8, 64, device="cuda")
    gy = torch.randn_like(x)

    def step():
        y, _ = m(x)
        return y.detach(), torch.autograd.grad(y, list(m.parameters()), gy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = step()
    torch.cuda.current_stream().wait_stream(side)
    del out
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, grads = step()
    runs = []
    for calls in (10, 11, 10):
        m.dropout.manual_seed(3, calls)
        graph.replay()
        runs.append((y.clone(), [g.clone() for g in grads]))
        assert m.dropout.key.tolist() == [3, calls + 1]
    assert not torch.equal(runs[0][0], runs[1][0])
    assert torch.equal(runs[0][0], runs[2][0])
    assert all(torch.equal(a, b) for a, b in zip(runs[0][1], runs[2][1]))
    m.dropout.manual_seed(3, 10)
    eager = step()
    assert torch.equal(eager[0], runs[0][0])


def test_block_dropout_in_the_model():
    torch.manual_seed(3)
    cfg = dict(input_dim=48, d_model=128, seq_len=16, num_layers=2, n_repeats=3, temporal=True, use_spikeskip=True,
               expansion=4)
    m = SpikingTransformer(**cfg, dropout=0.3, use_recurrence=True).cuda()
    ref = SpikingTransformer(**cfg, use_recurrence=True).cuda()
    ref.load_state_dict(m.state_dict())
    x = torch.randn(4, 16, 48, device="cuda")
    m.eval(), ref.eval()
    with torch.no_grad():  # dropout is off at inference: the same bits
        assert torch.equal(m(x), ref(x))
    m.train()
    logits = m(x)
    logits.square().sum().backward()
    for name, p in m.named_parameters():
        assert name.startswith(("exact_head", "embedding.temporal")) or p.grad is None or p.grad.isfinite().all(), name
    assert m.recurrence.vg_proj.weight.grad.abs().sum() > 0 and m.blocks[0].ffn.fc1.weight.grad.isfinite().all()
    with torch.no_grad():  # training mode without autograd drops too
        assert not torch.equal(m(x), m(x))
    assert m.blocks[0].drop_attn.key[1].item() == 3
    # a block's branches pass the dropout the operator defines
    blk = AstrocyteHebbianBlock(d_model=64, num_heads=4, dropout=0.4).cuda()
    blk.drop_attn.manual_seed(1), blk.drop_ffn.manual_seed(2)
    z = torch.randn(2, 3, 10, 64, device="cuda")
    out = blk(z)
    mid = ops.dropout(blk.attn(blk.norm1(z)), 0.4, (1, 0), residual=z)
    assert torch.equal(out, ops.dropout(blk.ffn(blk.norm2(mid)), 0.4, (2, 0), residual=mid))


def test_captured_inference_with_the_recurrence():
    torch.manual_seed(5)
    m = SpikingTransformer(input_dim=48, d_model=128, seq_len=16, n_repeats=70, temporal=True, use_spikeskip=True,
                           expansion=4, dropout=0.2, use_recurrence=True).cuda().eval()
    x = torch.randn(3, 16, 48, device="cuda")
    with torch.no_grad():
        fwd = CapturedForward(m, x)
        for _ in range(2):
            x = torch.randn(3, 16, 48, device="cuda")
            assert torch.equal(fwd(x).clone(), m(x))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_block_in_16_bits(dtype):
    torch.manual_seed(4)
    m = GatedRecurrence(64, groups=4, dropout=0.1).cuda().to(dtype)
    x = torch.randn(9, 2, 5, 64, device="cuda").to(dtype).requires_grad_()
    y, s = m(x)
    assert y.dtype == dtype and s.dtype == torch.float32
    y.float().square().sum().backward()
    assert all(p.grad is not None and p.grad.dtype == dtype and p.grad.isfinite().all() for p in m.parameters())
    m.eval()
    with torch.no_grad():
        want, last = m(x.detach())
        state = None
        for t in range(9):
            y, state = m.step(x[t].detach(), state)
            # one rounding of the projections' 16-bit results may fall the other way: a step of y's type
            assert (y - want[t]).abs().max() <= 4 * torch.finfo(dtype).eps * want.abs().max()


def test_refusals_and_autocast_branch():
    m = GatedRecurrence(32, groups=4).cuda()
    for bad in (torch.zeros(2, 3, 32, device="cuda"), torch.zeros(1, 2, 3, 16, device="cuda")):
        with pytest.raises(EngineError):
            m(bad)
    with pytest.raises(EngineError):
        m.step(torch.zeros(1, 2, 3, 32, device="cuda"))
    d = Dropout(0.5).cuda()
    x = torch.randn(100, device="cuda")
    d.manual_seed(4)
    want = ops.dropout(x.bfloat16().float(), 0.5, (4, 0), residual=x)
    assert torch.equal(d(x.bfloat16(), residual=x), want)  # a 16-bit branch on an fp32 residual
