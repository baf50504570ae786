"""GPU test: what the token-model operators write in place counts as written, so that a backward pass that has saved it refuses
instead of using the new values."""
import pytest
import torch

from distributed_tensorflow_amd.ops import embedding, muon, xent

pytestmark = pytest.mark.gpu


def _calls():
    ids, labels = torch.tensor([1, 3, 1], device="cuda"), torch.tensor([1, 0, -1], device="cuda")
    lr = torch.full((1,), 0.1, device="cuda")
    up = torch.ones(3, 5, device="cuda")

    def muon_step(t, which):
        rest = [torch.ones(3, 5, device="cuda") for _ in range(2)]
        muon.muon_step(muon.MuonPlan([t] if which == "w" else [rest[0]], [rest[1]], [rest[0]] if which == "w" else [t]), lr)

    return {"lookup": lambda t: embedding.lookup(torch.ones(7, 5, device="cuda"), ids, out=t),
            "lookup_grad": lambda t: embedding.lookup_grad(ids % 3, up, 3, out=t),
            "lookup_sgd": lambda t: embedding.lookup_sgd(t, ids % 3, up, lr),
            "xent, dz": lambda t: xent.sparse_softmax_xent_step(torch.zeros(3, 5, device="cuda"), labels, dz=t),
            "xent, logits": lambda t: xent.sparse_softmax_xent_step(t, labels, dz=t),
            "orthogonalize": lambda t: muon.orthogonalize(up, out=t),
            "orthogonalize, itself": lambda t: muon.orthogonalize(t, out=t),
            "weights": lambda t: muon_step(t, "w"), "momentum": lambda t: muon_step(t, "b")}


@pytest.mark.parametrize("name", ["lookup", "lookup_grad", "lookup_sgd", "xent, dz", "xent, logits", "orthogonalize",
                                  "orthogonalize, itself", "weights", "momentum"])
def test_a_saved_tensor_that_was_written_is_refused(name):
    x = torch.randn(3, 5, device="cuda", requires_grad=True)
    factor = torch.randn(3, 5, device="cuda")
    kept = factor.clone()
    out = x * factor                       # saves `factor`
    assert torch.equal(torch.autograd.grad(out.sum(), x, retain_graph=True)[0], kept)
    _calls()[name](factor)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out.sum(), x)


def test_the_loss_of_logits_that_became_their_gradient():
    z = torch.randn(4, 9, device="cuda", requires_grad=True)
    labels = torch.tensor([1, 0, -1, 8], device="cuda")
    loss = xent.sparse_softmax_xent(z, labels)
    xent.sparse_softmax_xent_step(z.detach(), labels, dz=z.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(loss.sum(), z)
