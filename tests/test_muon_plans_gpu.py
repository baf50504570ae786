"""GPU tests of what a MuonPlan keeps alive, and for how long."""
import pytest
import torch

from distributed_tensorflow_amd.ops import hip_backend as hb, muon

pytestmark = pytest.mark.gpu


def test_a_plan_dropped_while_its_step_is_under_way_on_a_side_stream():
    """Its workspace (and the tensors that it alone holds) are not given away before the side stream is done with them."""
    def make():
        shapes = [(300, 170), (170, 300)]
        ws = [torch.zeros(s, device="cuda") for s in shapes]
        gs = [torch.randn(s, device="cuda", generator=torch.Generator(device="cuda").manual_seed(i)) for i, s in enumerate(shapes)]
        return muon.MuonPlan(ws, gs, [torch.zeros(s, device="cuda") for s in shapes]), ws

    lr = torch.full((1,), 0.5, device="cuda")
    plan, want = make()
    muon.muon_step(plan, lr)
    del plan
    plan, got = make()
    torch.cuda.synchronize()
    held = [t for group in plan._groups for t in group if isinstance(t, torch.Tensor)] + plan.grads + plan.momenta
    places = [(t.numel() * t.element_size(), t.data_ptr()) for t in held]
    del held
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(5_000_000)
        muon.muon_step(plan, lr)
        done = side.record_event()
    del plan
    fresh = [torch.empty(n, dtype=torch.uint8, device="cuda") for n, _ in places]
    assert not done.query()              # (otherwise the allocator might have given the memory away rightly)
    assert not {t.data_ptr() for t in fresh} & {at for _, at in places}
    for t in fresh:
        t.fill_(255)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_learning_rate_that_the_step_would_write_is_refused():
    w, g, b = (torch.ones(8, 6, device="cuda") for _ in range(3))
    plan = muon.MuonPlan([w], [g], [b])
    for at in (w.view(-1)[:1], w.view(-1)[47:], b.view(-1)[5:6]):
        with pytest.raises(hb.HipKernelError):
            muon.muon_step(plan, at)
    assert bool((w == 1).all()) and bool((b == 1).all())
    muon.muon_step(plan, g.view(-1)[:1])            # (only read)
