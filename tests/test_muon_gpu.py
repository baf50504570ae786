"""GPU tests of the orthogonalised update (csrc/muon.hip) against the iteration in 64 bits.

Tolerance.  Every rounding of the kernels is at most 2^-22 of the value (two fp16 planes, and the dropped product of the low
planes) where that of an fp32 matrix product is 2^-24, the sums are fp32 in both, and what follows amplifies both alike: the
result is at most 4 times as far from the 64-bit iteration as the iteration in fp32 on the same input, measured here, plus one
2^-22 for each of the fifteen products and the input where that happens to be exact.  A store in bf16 / fp16 adds half a step."""
import math

import pytest
import torch

from distributed_tensorflow_amd.ops import hip_backend as hb, muon

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def factor(x, dtype=torch.float64, eps=muon.EPS):
    x = x.double()
    flip = x.shape[0] > x.shape[1]
    y = (x.t() if flip else x).contiguous()
    y = (y / (y.square().sum().sqrt() + eps)).to(dtype)
    a, b, c = muon.COEFFICIENTS
    for _ in range(muon.STEPS):
        p = y @ y.t().contiguous()
        y = a * y + (b * p + c * (p @ p)) @ y
    return y.t() if flip else y


def gradient(m, n, seed, noise=0.1):
    """A matrix with a few strong directions over noise."""
    g = gen(seed)
    r = max(1, min(m, n) // 8)
    return (torch.randn(m, r, device="cuda", generator=g) @ torch.randn(r, n, device="cuda", generator=g) / math.sqrt(r)
            + noise * torch.randn(m, n, device="cuda", generator=g))


def allowed(x, want):
    """Largest Frobenius distance from `want` that the note above allows."""
    return 4 * (factor(x, torch.float32).double() - want).norm() + 16 * 2.0 ** -22 * want.norm()


SHAPES = [(1, 1), (1, 7), (7, 1), (1, 300), (2, 3), (33, 65), (63, 64), (64, 64), (65, 63), (128, 128), (129, 127), (100, 784),
          (784, 100), (100, 10), (320, 1000), (1000, 320), (2050, 70), (512, 784), (1000, 1100), (1500, 1410), (1300, 2100)]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "%dx%d" % s)
@pytest.mark.parametrize("dtype", TYPES)
def test_factor_against_64_bits(shape, dtype):
    for noise in (1.0, 0.02):
        x = gradient(*shape, seed=sum(shape), noise=noise).to(dtype)
        want = factor(x)
        got = muon.orthogonalize(x)
        assert got.dtype == dtype and got.shape == x.shape
        tol = allowed(x, want) + (torch.finfo(dtype).eps / 2 * want.norm() if dtype != torch.float32 else 0)
        off = (got.double() - want).norm()
        assert float(off) <= float(tol), (float(off / want.norm()), float(tol / want.norm()))
        assert torch.equal(got, muon.orthogonalize(x))


@pytest.mark.parametrize("edge", [32, 64, 128, 192, 256])
@pytest.mark.parametrize("splits", [1, 2, 5])
def test_every_cut_of_the_products(edge, splits):
    """Tile edges and parts of k that the shapes alone would not choose: tiles that stick out on either side, parts without a
    step (a short matrix next to a long one), symmetric results with one and several tiles."""
    lib = hb.require()
    lib.dtf_debug_set_muon_cut(edge, splits)
    try:
        for shape in ((70, 130), (130, 900), (700, 520), (64, 64), (260, 2000)):
            x = gradient(*shape, seed=sum(shape))
            want = factor(x)
            assert float((muon.orthogonalize(x).double() - want).norm()) <= float(allowed(x, want)), shape
        shapes = [(30, 40), (500, 300), (64, 2000)]
        ws = [torch.zeros(s, device="cuda") for s in shapes]
        gs = [gradient(*s, seed=i) for i, s in enumerate(shapes)]
        muon.muon_step(muon.MuonPlan(ws, gs, [torch.zeros(s, device="cuda") for s in shapes]), torch.ones(1, device="cuda"),
                       momentum=0.0, nesterov=False)
        for w, g in zip(ws, gs):
            want = -math.sqrt(max(1.0, w.shape[1] / w.shape[0])) * factor(g)
            assert float((w.double() - want).norm()) <= math.sqrt(max(1.0, w.shape[1] / w.shape[0])) * float(allowed(g, factor(g)))
    finally:
        lib.dtf_debug_set_muon_cut(0, 0)


def test_layouts_and_in_place():
    room = torch.randn(300, 500, device="cuda", generator=gen(1))
    x = room[5:205, 3:133]
    before = room.clone()
    want = muon.orthogonalize(x.contiguous())
    assert torch.equal(muon.orthogonalize(x), want)
    muon.orthogonalize(x, out=x)
    assert torch.equal(x, want)
    room[5:205, 3:133] = before[5:205, 3:133]
    assert torch.equal(room, before)                   # nothing around the matrix was written
    turned = muon.orthogonalize(x.t().contiguous())     # the same iteration on the transpose
    assert float((turned.t() - want).norm()) <= 1e-6 * float(want.norm()) * 16


def test_zero_scale_and_what_is_not_finite():
    zero = torch.zeros(70, 130, device="cuda")
    assert torch.equal(muon.orthogonalize(zero), zero)
    x = gradient(70, 130, 2)
    want = muon.orthogonalize(x, eps=0.0)
    for power in (-60, 40):                            # the norm is formed in 64 bits: no scale under- or overflows
        assert torch.equal(muon.orthogonalize(x * 2.0 ** power, eps=0.0), want)
    spike = torch.zeros(64, 64, device="cuda")
    spike[3, 5] = -2.0                                 # rank one: the quintic of one singular value
    s = 1.0
    for _ in range(5):
        s = muon.COEFFICIENTS[0] * s + muon.COEFFICIENTS[1] * s ** 3 + muon.COEFFICIENTS[2] * s ** 5
    got = muon.orthogonalize(spike)
    assert abs(float(got[3, 5]) + s) < 1e-4 and int((got != 0).sum()) == 1
    for bad in (float("nan"), float("inf")):
        y = x.clone()
        y[3, 4] = bad
        assert bool(muon.orthogonalize(y).isnan().any())
    assert torch.equal(muon.orthogonalize(x, eps=0.0), want)      # and nothing of it stays behind


def test_singular_values_end_near_one():
    s = torch.linalg.svdvals(muon.orthogonalize(torch.randn(256, 1024, device="cuda", generator=gen(3))).double())
    assert 0.65 < float(s.min()) and float(s.max()) < 1.25         # the quintic's band for values above 0.01


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("shapes", [[(784, 100), (100, 10)], [(64, 64)], [(1, 9), (300, 200), (200, 300), (65, 1000)],
                                    [(40 + 7 * i, 90 - 5 * i) for i in range(11)], [(1400, 1300), (100, 60)]])
def test_step_against_64_bits(shapes, nesterov):
    ws = [torch.randn(s, device="cuda", generator=gen(10 + i)) for i, s in enumerate(shapes)]
    gs = [gradient(*s, seed=30 + i) for i, s in enumerate(shapes)]
    bs = [gradient(*s, seed=60 + i) for i, s in enumerate(shapes)]
    lr = torch.full((1,), 0.03, device="cuda")
    plan = muon.MuonPlan(ws, gs, bs)
    for step in range(2):
        w0, b0 = [w.double() for w in ws], [b.double() for b in bs]
        muon.muon_step(plan, lr, momentum=0.9, nesterov=nesterov)
        for w, g, b, w1, b1 in zip(ws, gs, bs, w0, b0):
            mu = float(torch.tensor(0.9))
            buf = mu * b1 + g.double()
            assert bool(((b.double() - buf).abs() <= 2.0 ** -24 * (2 * mu * b1.abs() + g.double().abs())).all())
            u = g + torch.tensor(0.9, device="cuda") * b if nesterov else b       # (the kernel's fp32 direction, to a rounding)
            k = float(lr) * math.sqrt(max(1.0, w.shape[1] / w.shape[0]))
            x = factor(u)
            # forming u rounds by 2^-24 of its terms; like any other perturbation of the input it ends up amplified by at most
            # 3.4445^5, the largest derivative of the quintic to the fifth
            slack = 3.4445 ** 5 * 2.0 ** -24 * float((g.abs() + 2 * b.abs()).norm() / u.norm())
            tol = k * (float(allowed(u, x)) + slack) + 2.0 ** -22 * float(w1.norm())
            assert float((w.double() - (w1 - k * x)).norm()) <= tol, step


def test_step_in_a_replayed_graph_and_on_a_side_stream():
    shapes = [(300, 170), (784, 512)]
    ws = [torch.randn(s, device="cuda", generator=gen(i)) for i, s in enumerate(shapes)]
    gs = [gradient(*s, seed=i) for i, s in enumerate(shapes)]
    bs = [torch.zeros(s, device="cuda") for s in shapes]
    lr = torch.full((1,), 0.02, device="cuda")
    plan = muon.MuonPlan(ws, gs, bs)
    start = [w.clone() for w in ws]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        muon.muon_step(plan, lr)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        muon.muon_step(plan, lr)
        factor_out = muon.orthogonalize(gs[0])
    for k in range(3):
        fresh = [gradient(*s, seed=100 + 10 * k + i) for i, s in enumerate(shapes)]
        results = []
        for eager in (False, True):
            for t, v in zip(ws + gs + bs, start + fresh + [torch.ones(s, device="cuda") * 0.01 for s in shapes]):
                t.copy_(v)
            lr.fill_(0.01 * (k + 1))
            if eager:
                muon.muon_step(plan, lr)
                f = muon.orthogonalize(gs[0])
            else:
                graph.replay()
                f = factor_out
            torch.cuda.synchronize()
            results.append([t.clone() for t in ws + bs + [f]])
        assert all(torch.equal(a, b) for a, b in zip(*results))


def test_refusals():
    w, g, b = (torch.zeros(8, 6, device="cuda") for _ in range(3))
    lr = torch.zeros(1, device="cuda")
    plan = muon.MuonPlan([w], [g], [b])
    bad = [lambda: muon.orthogonalize(w[0]), lambda: muon.orthogonalize(w.double()), lambda: muon.orthogonalize(w.t()),
           lambda: muon.orthogonalize(w[:0]), lambda: muon.orthogonalize(w, out=b[:7]), lambda: muon.orthogonalize(w, out=b.half()),
           lambda: muon.orthogonalize(w, eps=-1.0), lambda: muon.orthogonalize(w, eps=float("nan")),
           lambda: muon.MuonPlan([], [], []), lambda: muon.MuonPlan([w], [g], []), lambda: muon.MuonPlan([w], [g[:7]], [b]),
           lambda: muon.MuonPlan([w.half()], [g], [b]), lambda: muon.MuonPlan([w], [g], [w]), lambda: muon.MuonPlan([w], [w], [b]),
           lambda: muon.MuonPlan([w, w], [g, g], [b, b.clone()]), lambda: muon.MuonPlan([w[:, :4]], [g[:, :4]], [b[:, :4]]),
           lambda: muon.MuonPlan([w[0]], [g[0]], [b[0]]), lambda: muon.MuonPlan([w], [g.cpu()], [b]),
           lambda: muon.muon_step(plan, lr.double()), lambda: muon.muon_step(plan, torch.zeros(2, device="cuda")),
           lambda: muon.muon_step(plan, lr.cpu())]
    for k, call in enumerate(bad):
        with pytest.raises(hb.HipKernelError):
            call()
            pytest.fail(f"call {k} was not refused")


def test_a_plan_keeps_the_memory_it_was_made_on():
    w, g, b = torch.zeros(70, 40, device="cuda"), gradient(70, 40, seed=1), torch.zeros(70, 40, device="cuda")
    plan = muon.MuonPlan([w], [g], [b])
    want = -0.5 * muon.orthogonalize(g)
    w.data, g.data, b.data = (torch.ones(70, 40, device="cuda") for _ in range(3))
    muon.muon_step(plan, torch.full((1,), 0.5, device="cuda"), momentum=0.0)
    assert bool((w == 1).all()) and bool((g == 1).all()) and bool((b == 1).all())
    # (the same iteration on the same matrix; the update rounds once more, the halving does not)
    assert float((plan.params[0] - want).norm()) <= 2.0 ** -23 * float(want.norm())


def test_plans_on_two_streams_at_once():
    made = []
    for k in range(2):
        g = gradient(300, 500, seed=20 + k)
        made.append(([torch.zeros(300, 500, device="cuda")], [g], [torch.zeros(300, 500, device="cuda")]))
    lr = torch.full((1,), 0.25, device="cuda")
    want = []
    for ws, gs, bs in made:
        plan = muon.MuonPlan([w.clone() for w in ws], gs, [b.clone() for b in bs])
        for _ in range(5):
            muon.muon_step(plan, lr)
        want.append(plan.params[0])
    plans = [muon.MuonPlan(*m) for m in made]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for plan, s in zip(plans, streams):
            with torch.cuda.stream(s):
                muon.muon_step(plan, lr)
    torch.cuda.synchronize()
    assert all(torch.equal(p.params[0], x) for p, x in zip(plans, want))
