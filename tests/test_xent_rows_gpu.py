"""GPU test of more rows of logits than one native call takes.

Tolerance: three classes, so sums of three fp32 exponentials of values below 1: losses within 16 * 2^-24 of log 3 + 6 < 8, gradients
(at most the row's weight) within 16 * 2^-24 of it."""
import pytest
import torch

from distributed_tensorflow_amd.ops import xent

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [xent.LAUNCH_ROWS, 2 * xent.LAUNCH_ROWS + 5])
def test_more_rows_than_a_launch(rows):
    g = torch.Generator(device="cuda").manual_seed(rows)
    room = 2 * torch.randn(rows, 4, device="cuda", generator=g)
    z, labels = room[:, :3], torch.randint(-1, 4, (rows,), device="cuda", generator=g, dtype=torch.int32)
    weight = torch.rand(rows, device="cuda", generator=g)
    leaf = z.detach().requires_grad_(True)
    loss = xent.sparse_softmax_xent(leaf, labels)
    (got,) = torch.autograd.grad(loss, leaf, weight)
    logp = torch.log_softmax(z.double(), 1)
    at = labels.long().clamp(0, 2)[:, None]
    want = -logp.gather(1, at)[:, 0]
    dz = logp.exp().scatter_add(1, at, torch.full((rows, 1), -1.0, device="cuda", dtype=torch.float64))
    pad, wrong = labels < 0, labels > 2
    for t in (want, dz):
        t[pad] = 0
        t[wrong] = float("nan")

    def near(a, b, scale):
        assert torch.equal(a.isnan(), b.isnan())
        assert float((a.double() - b).nan_to_num().abs().max()) <= 16 * 2.0 ** -24 * scale

    near(loss.detach(), want, 8)
    near(got, dz * weight.double()[:, None], 1)
    step_dz = torch.empty(rows, 3, device="cuda")
    near(xent.sparse_softmax_xent_step(z, labels, dz=step_dz, grad_scale=0.5), want, 8)
    near(step_dz, 0.5 * dz, 1)
    before = room[:, 3].clone()
    xent.sparse_softmax_xent_step(z, labels, dz=z, grad_scale=0.5)
    assert torch.equal(z.nan_to_num(), step_dz.nan_to_num()) and torch.equal(room[:, 3], before)
