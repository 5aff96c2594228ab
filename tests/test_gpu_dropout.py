"""Counter-based dropout (spk_dropout): the mask bit for bit against Philox4x32
with 7 rounds in Python integers, values to rounding, its backward pass, and
its keys on host and device."""
import pytest
import torch

from spikestack_lite_b200 import ops
from spikestack_lite_b200._lib import EngineError
from tests.temporal_ref import U, assert_within, dropout_words, philox, stored

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
KEYS = [(0, 0), (0x0123456789ABCDEF, 7), ((1 << 64) - 1, 0xFEDCBA9876543210)]


def mask(n, p, key):
    return torch.tensor([w >= int(p * 2.0 ** 32 + 0.5) for w in dropout_words(n, *key)], dtype=torch.bool)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("n", [1, 3, 4, 5, 8, 31, 257, 4099])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 0.999, 1.0])
def test_matches_the_generator(n, p, dtype):
    g = torch.Generator().manual_seed(n)
    x, r, gy = (torch.randn(n, generator=g).to(DT[dtype]) for _ in range(3))
    for key in KEYS[:1] if n > 1000 else KEYS:
        keep = mask(n, p, key)
        scale = 1.0 / (1.0 - p) if p < 1 else 0.0
        for res in (None, r):
            xd = x.cuda().requires_grad_()
            rd = None if res is None else res.cuda().requires_grad_()
            y = ops.dropout(xd, p, key, residual=rd)
            kept = torch.where(keep, x.double() * scale, 0.0)
            want = kept + (0.0 if res is None else res.double())
            # the scale's and the product's rounding, then the sum's
            assert_within(y, want, stored(2 * U * kept.abs() + U * want.abs(), want, DT[dtype]), "y")
            ins = (xd,) if res is None else (xd, rd)
            grads = torch.autograd.grad(y, ins, gy.cuda())
            gx = torch.where(keep, gy.double() * scale, 0.0)
            assert_within(grads[0], gx, stored(2 * U * gx.abs(), gx, DT[dtype]), "gx")
            if res is not None:
                assert torch.equal(grads[1].cpu(), gy)
            ones = torch.ones(n, dtype=DT[dtype], device="cuda")
            assert torch.equal(ops.dropout(ones, p, key) != 0, keep.cuda() if p < 1 else torch.zeros_like(keep).cuda())


def test_device_keys_equal_host_keys_and_misaligned_views():
    base = torch.randn(1031, device="cuda")
    for key in KEYS:
        signed = [v - (1 << 64) if v >= 1 << 63 else v for v in key]
        dev = torch.tensor(signed, dtype=torch.int64, device="cuda")
        want = ops.dropout(base[:1030].clone(), 0.3, key)
        assert torch.equal(ops.dropout(base[:1030].clone(), 0.3, dev), want)
        assert torch.equal(ops.dropout(base[:1030].clone(), 0.3, signed), want)
        for dt in DT.values():  # the mask goes by the element's index, not by its address
            src = torch.zeros(1031, dtype=dt, device="cuda")
            src[1:] = base[:1030].to(dt)
            assert torch.equal(ops.dropout(src[1:], 0.3, key), ops.dropout(src[1:].clone(), 0.3, key))
            assert torch.equal(ops.dropout(src[1:], 0.3, key, residual=src[1:].clone()),
                               ops.dropout(src[1:].clone(), 0.3, key, residual=src[1:].clone()))


def test_rate_and_independence():
    n, p = 1 << 22, 0.1
    ones = torch.ones(n, device="cuda")
    a = ops.dropout(ones, p, (1, 0)) != 0
    for other in ((1, 1), (2, 0), (1 << 33, 0), (1, 1 << 40)):
        b = ops.dropout(ones, p, other) != 0
        # kept by both: binomial with 0.81; 6 standard deviations
        both = (a & b).double().mean().item()
        assert abs(both - 0.81) < 6 * (0.81 * 0.19 / n) ** 0.5
        assert abs(b.double().mean().item() - 0.9) < 6 * (0.09 / n) ** 0.5
    # neighbours are independent: both dropped with 0.01
    for lag in (1, 2, 3, 4, 512):
        pair = (~a[lag:] & ~a[:-lag]).double().mean().item()
        assert abs(pair - 0.01) < 6 * (0.01 / n) ** 0.5


def test_masked_non_finite_values_and_non_contiguous_inputs():
    n = 1000
    keep = mask(n, 0.5, (3, 4)).cuda()
    x = torch.randn(n, device="cuda")
    y = ops.dropout(torch.where(keep, x, float("nan")), 0.5, (3, 4))
    assert torch.equal(y, torch.where(keep, 2 * x, 0.0))
    y = ops.dropout(torch.where(keep, x, float("inf")), 0.5, (3, 4), residual=x)
    assert y.isfinite().all()
    m = torch.randn(20, 50, device="cuda")
    assert torch.equal(ops.dropout(m.t(), 0.5, (3, 4)), ops.dropout(m.t().contiguous(), 0.5, (3, 4)))
    assert ops.dropout(torch.empty(0, 3, device="cuda"), 0.5, (3, 4)).shape == (0, 3)


def test_a_captured_graph_takes_the_keys_of_its_replay():
    x = torch.randn(4096, device="cuda")
    gy = torch.randn(4096, device="cuda")
    key = torch.tensor([11, 0], dtype=torch.int64, device="cuda")

    def train():
        xd = x.detach().requires_grad_()
        y = ops.dropout(xd, 0.2, key)
        return y.detach(), torch.autograd.grad(y, xd, gy)[0]

    train()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, gx = train()
    for off in (0, 5):
        key[1] = off
        graph.replay()
        assert torch.equal(y, ops.dropout(x, 0.2, (11, off)))
        assert torch.equal(gx, ops.dropout(gy, 0.2, (11, off)))
    # a key that changes between forward and backward is refused, not silently used
    xd = x.detach().requires_grad_()
    out = ops.dropout(xd, 0.2, key)
    key[1] += 1
    with pytest.raises(RuntimeError):
        torch.autograd.grad(out, xd, gy)


def test_offsets_beyond_32_bits():
    n = (1 << 31) + 6
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    y = ops.dropout(x, 0.5, (9, 1 << 35))
    for start in (0, (1 << 31) - 8, n - 10):
        first = start // 4
        words = []
        for i in range(first, first + 4):
            words += philox((i & 0xFFFFFFFF, i >> 32, 0, (1 << 35) >> 32), (9, 0))
        keep = torch.tensor([w >= 1 << 31 for w in words])[start - 4 * first:][:min(10, n - start)]
        assert torch.equal(y[start:start + len(keep)].float().cpu(), 2.0 * keep.float())


def test_no_second_derivative():
    x = torch.randn(8, device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad(ops.dropout(x, 0.5, (0, 0)).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_refusals():
    x = torch.randn(4, 8, device="cuda")
    for args in ((x, -0.1, (0, 0)), (x, 1.1, (0, 0)), (x, float("nan"), (0, 0)), (x.double(), 0.1, (0, 0)),
                 (x, 0.1, 5), (x, 0.1, (1, 2, 3)), (x, 0.1, torch.zeros(2, dtype=torch.int64)),
                 (x, 0.1, torch.zeros(2, device="cuda")), (x, 0.1, torch.zeros(3, dtype=torch.int64, device="cuda"))):
        with pytest.raises(EngineError):
            ops.dropout(*args)
    for r in (x[:2], x.half(), x.cpu()):
        with pytest.raises(EngineError):
            ops.dropout(x, 0.1, (0, 0), residual=r)
