"""GPU tests of the orthogonalised update in rows and columns that are little next to the others (a feature hardly seen).

Tolerance.  The kernels keep every entry to 2^-22 of the largest one that its own row (or column) may have and sum in fp32, where fp32
matrix products round to 2^-24 of each term; what follows amplifies both alike.  So the part of the result that lies in such rows is
at most 4 times as far from the 64-bit iteration as that part of the iteration in fp32, measured here, plus one 2^-22 for each of the
fifteen products and the input where that happens to be exact; the whole result too."""
import math

import pytest
import torch

from distributed_tensorflow_amd.ops import hip_backend as hb, muon

pytestmark = pytest.mark.gpu


def factor(x, dtype=torch.float64):
    """(In fp32 the norm is still formed in 64 bits.)"""
    x = x.double()
    flip = x.shape[0] > x.shape[1]
    y = (x.t() if flip else x).contiguous()
    y = (y / (y.square().sum().sqrt() + muon.EPS)).to(dtype)
    a, b, c = muon.COEFFICIENTS
    for _ in range(muon.STEPS):
        p = y @ y.t().contiguous()
        y = a * y + (b * p + c * (p @ p)) @ y
    return y.t() if flip else y


def matrix(shape, kind, scale, seed=0):
    """The matrix and a mask of its little part."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, device="cuda", generator=g)
    i, j = torch.arange(shape[0], device="cuda")[:, None], torch.arange(shape[1], device="cuda")[None]
    if kind == "both":
        x = x * torch.where(i % 2 == 0, scale, 1.0) * torch.where(j % 3 == 0, scale, 1.0)
        return x, (i % 2 == 0) | (j % 3 == 0)
    little = {"rows": (i % 2 == 0) & (j >= 0), "columns": (j % 2 == 0) & (i >= 0), "one row": (i == shape[0] // 2) & (j >= 0),
              "spikes": ~((i % 7 == 0) & (j % 5 == 0))}[kind]
    x = torch.where(little, x * scale, x)
    return x, (i % 7 != 0) & (j >= 0) if kind == "spikes" else little         # (of the spikes: the rows without one)


def check(got, x, little):
    want, plain = factor(x), factor(x, torch.float32).double()
    for part in (little, ~little, torch.ones_like(little)):
        w = want[part]
        off, allowed = (got.double()[part] - w).norm(), 4 * (plain[part] - w).norm() + 16 * 2.0 ** -22 * w.norm()
        assert float(off) <= float(allowed), (float(off / w.norm()), float(allowed / w.norm()))


@pytest.mark.parametrize("kind", ["rows", "columns", "both", "one row", "spikes"])
@pytest.mark.parametrize("scale", [1e-3, 1e-6, 1e-9, 1e-14])
def test_little_rows_and_columns(kind, scale):
    for k, shape in enumerate(((256, 512), (300, 70), (65, 1000), (520, 520), (1100, 1000))):
        x, little = matrix(shape, kind, scale, k)
        got = muon.orthogonalize(x)
        check(got, x, little)
        assert torch.equal(got, muon.orthogonalize(x))


@pytest.mark.parametrize("edge", [32, 64, 128, 192, 256])
@pytest.mark.parametrize("splits", [1, 3])
def test_little_rows_under_every_cut(edge, splits):
    lib = hb.require()
    lib.dtf_debug_set_muon_cut(edge, splits)
    try:
        for kind in ("rows", "both"):
            for shape in ((300, 900), (700, 410)):
                x, little = matrix(shape, kind, 1e-8)
                check(muon.orthogonalize(x), x, little)
    finally:
        lib.dtf_debug_set_muon_cut(0, 0)


def test_little_rows_of_16_bit_matrices():
    for dtype, scale in ((torch.bfloat16, 1e-10), (torch.float16, 1e-4)):
        x, little = matrix((256, 512), "rows", scale)
        x = x.to(dtype)
        want, got = factor(x), muon.orthogonalize(x)
        # half a step of the type (of its smallest normal value where the result is below that), behind the fp32 result's own bound
        step = torch.finfo(dtype).eps / 2 * want.abs().clamp(min=torch.finfo(dtype).tiny)
        off = ((got.double() - want).abs() - step).clamp(min=0)[little]
        plain = (factor(x, torch.float32).double() - want)[little]
        assert float(off.norm()) <= 4 * float(plain.norm()) + 16 * 2.0 ** -22 * float(want[little].norm())


def test_little_rows_in_a_step():
    """The weights start at zero, so that the update itself is what is stored; two matrices of one plan."""
    made = [matrix((200, 500), "rows", 1e-9, 1), matrix((500, 130), "columns", 1e-7, 2)]
    ws = [torch.zeros_like(x) for x, _ in made]
    plan = muon.MuonPlan(ws, [x for x, _ in made], [torch.zeros_like(x) for x, _ in made])
    muon.muon_step(plan, torch.full((1,), -1.0, device="cuda"), momentum=0.0, nesterov=False)
    for w, (x, little) in zip(ws, made):
        check(w / math.sqrt(max(1.0, x.shape[1] / x.shape[0])), x, little)


def test_zeros_and_lengths():
    """Rows and columns of zeros stay zeros; a matrix of zeros does without eps too; one row or column is scaled to the quintic's value
    whatever its length."""
    for shape in ((1, 1), (64, 64), (70, 130)):
        zero = torch.zeros(shape, device="cuda")
        assert torch.equal(muon.orthogonalize(zero, eps=0.0), zero)
    x = torch.randn(90, 200, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5))
    x[::3] = 0
    x[:, 50:120] = 0
    got = muon.orthogonalize(x)
    assert bool((got[::3] == 0).all()) and bool((got[:, 50:120] == 0).all())
    check(got, x, x != 0)
    s = 1.0
    for _ in range(muon.STEPS):
        s = muon.COEFFICIENTS[0] * s + muon.COEFFICIENTS[1] * s ** 3 + muon.COEFFICIENTS[2] * s ** 5
    for n in (1, 63, 4097, 65536):
        row = torch.randn(1, n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(n))
        for x in (row, row.t().contiguous()):
            # the one singular value takes the scalar iteration, in fp32: at most 485 times 16 roundings
            got = muon.orthogonalize(x, eps=0.0).double()
            want = s * x.double() / x.double().norm()
            assert float((got - want).norm()) <= 485 * 16 * 2.0 ** -24


def test_a_matrix_far_below_eps():
    x, little = matrix((150, 90), "rows", 1e-6)
    check(muon.orthogonalize(x * 1e-20), x * 1e-20, little)
