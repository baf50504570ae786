"""CPU tests of the token-model operators: what the native entry points and the wrappers refuse before anything is launched,
and the torch paths that CPU tensors take (same rules as the kernels)."""
import math

import pytest
import torch

from distributed_tensorflow_amd.ops import embedding, hip_backend as hb, xent

SHAPE, NULL = 1, 2


def test_native_refusals_of_the_lookup():
    lib = hb.require()
    one = 4096      # a non-null address that nothing dereferences: every call below is refused on the host
    call = lambda rows=4, dim=8, ld=8, tokens=3, ldo=8, dtype=0, t=one, i=one, o=one: lib.dtf_embed_lookup(  # noqa: E731
        t, dtype, rows, dim, ld, i, 1, tokens, 1.0, o, ldo, None)
    assert call(rows=0) == call(dim=0) == call(ld=7) == call(ldo=7) == call(tokens=-1) == call(dtype=3) == call(dtype=-1) == SHAPE
    assert call(tokens=(1 << 26) + 1) == call(rows=(1 << 28) + 1) == call(dim=(1 << 20) + 1, ld=1 << 21, ldo=1 << 21) == SHAPE
    assert call(t=None) == call(i=None) == call(o=None) == NULL
    assert call(tokens=0) == 0


def test_native_refusals_of_the_gradient_and_the_row_update():
    lib = hb.require()
    one, need = 4096, lib.dtf_embed_workspace(3, 8)
    assert need > 0 and lib.dtf_embed_workspace(-1, 8) == lib.dtf_embed_workspace(3, 0) == -1

    def grad(rows=4, dim=8, ldg=8, ldt=8, tokens=3, dtype=0, i=one, g=one, o=one, ws=one, size=need):
        return lib.dtf_embed_grad(i, 1, tokens, g, ldg, o, dtype, rows, dim, ldt, 1.0, ws, size, None)

    assert grad(rows=0) == grad(dim=0) == grad(ldg=7) == grad(ldt=7) == grad(tokens=-1) == grad(dtype=3) == SHAPE
    assert grad(size=need - 1) == grad(ws=one + 4) == SHAPE
    assert grad(i=None) == grad(g=None) == grad(o=None) == grad(ws=None) == NULL

    def sgd(tokens=3, lr=one, ws=one, size=need):
        return lib.dtf_embed_sgd(one, 1, tokens, one, 8, one, 0, 4, 8, 8, 1.0, lr, ws, size, None)

    assert sgd(lr=None) == NULL and sgd(size=0) == SHAPE and sgd(tokens=0) == 0


def test_native_refusals_of_the_cross_entropy():
    lib = hb.require()
    one = 4096

    def step(tokens=3, classes=8, ld=8, dtype=0, z=one, lab=one, dz=one, ldz=8):
        return lib.dtf_sparse_xent(z, dtype, tokens, classes, ld, lab, 1, dz, ldz, 1.0, one, None, None)

    assert step(classes=0) == step(ld=7) == step(ldz=7) == step(tokens=-1) == step(dtype=3) == step(tokens=(1 << 21) + 1) == SHAPE
    assert step(classes=(1 << 26) + 1, ld=1 << 27, ldz=1 << 27) == SHAPE
    assert step(z=None) == step(lab=None) == NULL and step(tokens=0) == 0

    def back(stats=one, g=one, dz=one):
        return lib.dtf_sparse_xent_grad(one, 0, 3, 8, 8, one, 1, stats, g, 1, dz, 8, None)

    assert back(stats=None) == back(g=None) == back(dz=None) == NULL


def test_wrappers_refuse_cpu_tensors():
    t, i, lr = torch.zeros(4, 8), torch.zeros(3, dtype=torch.long), torch.zeros(1)
    for call in (lambda: embedding.lookup(t, i), lambda: embedding.lookup_grad(i, t[:3], 4),
                 lambda: embedding.lookup_sgd(t, i, t[:3], lr), lambda: xent.sparse_softmax_xent_step(t[:3], i)):
        with pytest.raises(hb.HipKernelError):
            call()


def test_lookup_on_the_cpu():
    table = torch.randn(6, 4, dtype=torch.float64, requires_grad=True)
    ids = torch.tensor([[5, 0], [-1, 6], [5, 2]])
    out = embedding.embedding_lookup(table, ids, 2.0)
    assert torch.equal(out[0, 0], 2 * table[5]) and bool((out[1] == 0).all()) and out.shape == (3, 2, 4)
    (g,) = torch.autograd.grad(out.sum(), table)
    assert g[:, 0].tolist() == [2, 0, 2, 0, 0, 4]
    assert torch.autograd.gradcheck(lambda t: embedding.embedding_lookup(t, ids, 1.5), table)


def test_cross_entropy_on_the_cpu():
    z = torch.randn(6, 5, requires_grad=True)
    labels = torch.tensor([0, 4, -1, 2, 5, -7])
    loss = xent.sparse_softmax_xent(z, labels)
    want = torch.nn.functional.cross_entropy(z, labels.clamp(0, 4), reduction="none")
    ok = torch.tensor([0, 1, 3])
    assert torch.allclose(loss[ok], want[ok]) and loss[2] == 0 and loss[5] == 0 and math.isnan(float(loss[4]))
    (g,) = torch.autograd.grad(loss, z, torch.ones(6))
    (w,) = torch.autograd.grad(want, z, torch.ones(6))
    assert torch.allclose(g[ok], w[ok]) and bool((g[2] == 0).all()) and bool((g[5] == 0).all()) and bool(g[4].isnan().all())
    with torch.no_grad():
        z[2] = float("nan")                 # padding is not looked at
        z[0, 1:] = -float("inf")
    loss = xent.sparse_softmax_xent(z, labels)
    (g,) = torch.autograd.grad(loss, z, torch.ones(6))
    assert loss[2] == 0 and bool((g[2] == 0).all()) and loss[0] == 0 and bool((g[0] == 0).all()) and torch.allclose(g[3], w[3])


def test_native_refusals_of_the_orthogonalised_update():
    import ctypes as C

    from distributed_tensorflow_amd.ops import muon

    lib = hb.require()
    one = 4096
    r, c = (C.c_int32 * 9)(*[8] * 9), (C.c_int32 * 9)(*[6] * 9)
    need = lib.dtf_muon_workspace(1, r, c)
    assert need > 0 and lib.dtf_muon_workspace(0, r, c) == lib.dtf_muon_workspace(9, r, c) == lib.dtf_muon_workspace(1, None, c) == -1
    assert lib.dtf_muon_workspace(1, (C.c_int32 * 1)(0), c) == lib.dtf_muon_workspace(1, (C.c_int32 * 1)(1 << 17), c) == -1

    def factor(dtype=0, rows=8, cols=6, ldx=6, ldo=6, eps=0.0, x=one, o=one, ws=one, size=need):
        return lib.dtf_orthogonalize(x, dtype, rows, cols, ldx, o, ldo, eps, ws, size, None)

    assert factor(dtype=3) == factor(rows=0) == factor(cols=0) == factor(ldx=5) == factor(ldo=5) == factor(eps=-1.0) == SHAPE
    assert factor(eps=float("nan")) == factor(size=need - 1) == factor(ws=one + 16) == SHAPE
    assert factor(x=None) == factor(o=None) == factor(ws=None) == NULL
    p = (C.c_uint64 * 9)(*[one] * 9)
    null = (C.c_uint64 * 9)()

    def step(n=1, w=p, g=p, b=p, lr=one, eps=0.0, ws=one, size=need):
        return lib.dtf_muon_step(n, r, c, w, g, b, lr, 0.9, 1, eps, ws, size, None)

    assert step(n=0) == step(n=9) == step(eps=-1.0) == step(size=need - 1) == step(ws=one + 16) == SHAPE
    assert step(w=None) == step(lr=None) == step(ws=None) == step(w=null) == step(g=null) == step(b=null) == NULL
    with pytest.raises(hb.HipKernelError):
        muon.orthogonalize(torch.zeros(3, 4))
    with pytest.raises(hb.HipKernelError):
        muon.MuonPlan([torch.zeros(3, 4)], [torch.zeros(3, 4)], [torch.zeros(3, 4)])


def test_native_refusals_of_few_long_rows():
    lib = hb.load()
    need = lib.dtf_sparse_xent_workspace(0, 3, 300000)
    assert need > 0 and lib.dtf_sparse_xent_workspace(0, 65, 300000) == 0 and lib.dtf_sparse_xent_workspace(0, 3, 300) == 0
    assert lib.dtf_sparse_xent_workspace(3, 3, 300000) < 0 and lib.dtf_sparse_xent_workspace(0, -1, 300000) < 0
    assert lib.dtf_sparse_xent_workspace(0, 3, (1 << 26) + 1) < 0 and lib.dtf_sparse_xent_workspace(0, 3, 0) < 0
    one = 4096

    def step(ws=one, size=need, dtype=0, ld=300000):
        return lib.dtf_sparse_xent_cut(one, dtype, 3, 300000, ld, one, 1, one, 300000, 1.0, one, None, ws, size, None)

    assert step(size=need - 1) == step(ws=one + 4) == step(dtype=3) == step(ld=299999) == SHAPE
