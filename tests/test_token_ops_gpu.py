"""GPU tests of the token-model operators (csrc/embed.hip, csrc/xent.hip) against plain 64-bit implementations.

Tolerances.  A sum of n fp32 terms is off by at most (n + 1) 2^-24 sum|terms| (each product and each addition rounds by half a
step); a store in type t adds eps_t / 2 of the value (or half a subnormal step).  An exponential of the cross-entropy is off by
2^-24 (4 + 3 |z - max|): the subtraction, the multiplication by log2(e) and its constant each move the exponent by half a step
of |z - max|, the exponential itself is good to one step; a row's sum adds the additions of one thread and of the exchange."""
import math

import pytest
import torch

from distributed_tensorflow_amd.ops import embedding, hip_backend as hb, xent

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(t, value):
    return torch.finfo(t).eps / 2 * value.abs() + torch.finfo(t).smallest_normal * torch.finfo(t).eps


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def make_ids(tokens, rows, seed, pad=0.1, kind="words"):
    g = gen(seed)
    if kind == "words":
        u = torch.rand(tokens, device="cuda", generator=g, dtype=torch.float64)
        ids = (torch.exp(u * math.log(rows + 1)) - 1).long().clamp_(0, rows - 1)
    elif kind == "uniform":
        ids = torch.randint(0, rows, (tokens,), device="cuda", generator=g)
    elif kind == "one":
        ids = torch.full((tokens,), rows - 1, device="cuda")
    else:
        ids = torch.full((tokens,), -1, device="cuda")
    if pad and kind != "one":
        r = torch.rand(tokens, device="cuda", generator=g)
        ids[r < pad] = -1
        ids[r < pad / 2] = rows           # past the end: padding as well
    return ids


def exact_sums(ids, g, rows):
    """(sum, sum of magnitudes, count) by row in 64 bits."""
    ok = (ids >= 0) & (ids < rows)
    total = torch.zeros(rows + 1, g.shape[1], device="cuda", dtype=torch.float64)
    size = torch.zeros_like(total)
    at = torch.where(ok, ids.long(), rows)
    total.index_add_(0, at, g.double())
    size.index_add_(0, at, g.double().abs())
    return total[:rows], size[:rows], torch.bincount(at, minlength=rows + 1)[:rows]


# tokens around a chunk, the largest number that is compared in pairs, a block of the multi-block sort, and more than one of its tiles
TOKENS = [0, 1, 2, 31, 64, 65, 1000, 4095, 4096, 4097, 9001, 140001]
DIMS = [1, 3, 8, 101, 256, 257, 1030]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", TOKENS)
@pytest.mark.parametrize("dim", [1, 7, 64, 101, 1024, 2056])
def test_lookup_is_the_scaled_row(dtype, tokens, dim):
    rows = 517
    table = torch.randn(rows, dim, device="cuda", generator=gen(1)).to(dtype)
    ids = make_ids(tokens, rows, 2)
    got = embedding.lookup(table, ids, 1.7)
    ok = (ids >= 0) & (ids < rows)
    want = table[torch.where(ok, ids, 0)].double() * float(torch.tensor(1.7))
    want[~ok] = 0
    # the fp32 product rounds by U, its store by half a step; for fp16 the hardware rounds the exact product to fp16 at once
    # (one instruction multiplies and converts), which is within half a step of it: the same bound covers both
    assert got.shape == (tokens, dim)
    assert bool(((got.double() - want).abs() <= half_step(dtype, want) * (1 + U) + U * want.abs()).all())
    assert bool((got[~ok] == 0).all())
    assert torch.equal(embedding.lookup(table, ids.int(), 1.7), got)


@pytest.mark.parametrize("dtype", TYPES)
def test_lookup_strides_and_out(dtype):
    wide = torch.randn(40, 50, device="cuda", generator=gen(3)).to(dtype)
    table = wide[:, 3:40]                                        # rows apart, unaligned
    ids = torch.tensor([[0, 39, 7], [-1, 40, 7]], device="cuda")
    got = embedding.lookup(table, ids, 0.5)
    want = (table[ids.clamp(0, 39)].float() * 0.5).to(dtype)
    want[1, :2] = 0
    assert got.shape == (2, 3, 37) and torch.equal(got, want)
    room = torch.full((8, 45), 9.0, device="cuda").to(dtype)
    embedding.lookup(table, ids, 0.5, out=room[1:7, 2:39])
    assert torch.equal(room[1:7, 2:39], want.view(6, 37))
    assert bool((room[0] == 9).all() and (room[7] == 9).all() and (room[:, :2] == 9).all() and (room[:, 39:] == 9).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", TOKENS)
@pytest.mark.parametrize("kind", ["words", "uniform", "one", "padding"])
def test_gradient_against_64_bits(dtype, tokens, kind):
    for rows, dim in ((1, 5), (777, 101), (300, 256)):
        ids = make_ids(tokens, rows, 4, kind=kind)
        g = torch.randn(tokens, dim, device="cuda", generator=gen(5)).to(dtype)
        if dtype == torch.float16:
            g = g / 64                   # (sums of 140001 equal signs stay below 65504)
        got = embedding.lookup_grad(ids, g, rows, 1.5)
        total, size, count = exact_sums(ids, g, rows)
        tol = (count[:, None] + 3) * U * 1.5 * size + half_step(dtype, 1.5 * total)
        assert got.dtype == dtype and got.shape == (rows, dim)
        assert bool(((got.double() - 1.5 * total).abs() <= tol).all()), (rows, dim)
        assert bool((got[count == 0] == 0).all())
        again = embedding.lookup_grad(ids.int(), g, rows, 1.5)
        assert torch.equal(got, again)               # the order of additions does not change from run to run


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("tokens", [1, 100, 4097, 30000])
def test_row_update_touches_what_occurs(dtype, dim, tokens):
    rows, lr, scale = 1009, 0.25, 1.25
    room = torch.randn(rows + 2, dim + 3, device="cuda", generator=gen(6)).to(dtype)
    before = room.clone()
    table = room[1:rows + 1, 2:dim + 2]
    ids = make_ids(tokens, rows, 7, kind="words")
    g = (torch.randn(tokens, dim, device="cuda", generator=gen(8)) / 16).to(dtype)
    out = embedding.lookup_sgd(table, ids, g, torch.full((1,), lr, device="cuda"), scale)
    assert out is table
    total, size, count = exact_sums(ids, g, rows)
    old = before[1:rows + 1, 2:dim + 2].double()
    want = old - lr * scale * total
    # the factor lr * scale and its product round, then the subtraction (of the exact table value), then the store
    tol = (count[:, None] + 4) * U * lr * scale * size + U * (old.abs() + lr * scale * size) + half_step(dtype, want)
    assert bool(((table.double() - want).abs() <= tol).all())
    assert torch.equal(table[count == 0], before[1:rows + 1, 2:dim + 2][count == 0])
    room[1:rows + 1, 2:dim + 2] = before[1:rows + 1, 2:dim + 2]
    assert torch.equal(room, before)                 # nothing around the table was written


def test_gradient_layouts_of_the_upstream_gradient():
    ids = make_ids(500, 50, 9)
    wide = torch.randn(500, 90, device="cuda", generator=gen(10))
    for g in (wide[:, 5:69], wide.t()[:64, :].t(), wide[:1, :64].expand(500, 64)):
        total, size, count = exact_sums(ids, g, 50)
        got = embedding.lookup_grad(ids, g, 50)
        assert bool(((got.double() - total).abs() <= (count[:, None] + 3) * U * size + half_step(torch.float32, total)).all())


def test_gradient_carries_infinities_and_nan_to_their_rows_only():
    ids = torch.tensor([3, 1, 3, -1, 5, 1], device="cuda")
    g = torch.ones(6, 8, device="cuda")
    g[0, 2], g[3], g[4, 1] = float("inf"), float("nan"), float("nan")
    got = embedding.lookup_grad(ids, g, 7)
    want = torch.zeros(7, 8, device="cuda")
    want[3], want[1], want[5] = 2.0, 2.0, 1.0
    want[3, 2], want[5, 1] = float("inf"), float("nan")
    assert torch.equal(torch.nan_to_num(got, 5.5, 6.5), torch.nan_to_num(want, 5.5, 6.5))


def test_offsets_past_32_bits():
    """A table of 2^31 + elements: the last rows are read, summed and updated where they are."""
    rows, dim = (1 << 19) + 7, 4100
    table = torch.zeros(rows, dim, device="cuda", dtype=torch.bfloat16)
    table[-1], table[-2], table[0] = 3.0, 2.0, 1.0
    ids = torch.tensor([rows - 1, 0, rows - 2, rows], device="cuda")
    got = embedding.lookup(table, ids)
    assert got[:, 0].tolist() == [3, 1, 2, 0] and got[:, -1].tolist() == [3, 1, 2, 0]
    g = torch.ones(4, dim, device="cuda", dtype=torch.bfloat16)
    embedding.lookup_sgd(table, ids, g, torch.ones(1, device="cuda"))
    assert table[[0, rows - 2, rows - 1], -1].tolist() == [0, 1, 2] and float(table.float().abs().sum()) == 3 * dim
    grad = embedding.lookup_grad(ids, g, rows)
    assert float(grad.float().sum()) == 3 * dim and grad[rows - 1, -1] == 1 and grad[rows - 3, -1] == 0


def test_lookup_through_autograd_and_differences():
    table = torch.randn(11, 5, device="cuda", generator=gen(11)).requires_grad_(True)
    ids = torch.tensor([[1, 10, 1], [-1, 0, 11]], device="cuda")
    w = torch.randn(2, 3, 5, device="cuda", generator=gen(12))

    def f(t):
        return (torch.tanh(embedding.embedding_lookup(t, ids, 3.0)) * w).sum()

    (got,) = torch.autograd.grad(f(table), table)
    h = 2.0 ** -9
    with torch.no_grad():
        for v, c in ((1, 0), (10, 4), (0, 2), (5, 1)):
            e = torch.zeros_like(table)
            e[v, c] = h
            # central differences of an fp32 function: truncation h^2 |f'''| / 6 <= h^2 * 2 * 27 * |w| n / 6 (n <= 2 occurrences,
            # |w| < 4), rounding of the two sums of 30 terms below 4: 30 * 30 * 4 * 2^-24 / h
            diff = (f(table + e) - f(table - e)) / (2 * h)
            assert abs(float(diff - got[v, c])) <= h * h * 2 * 27 * 4 * 2 / 6 + 30 * 30 * 4 * U / h
    (ones,) = torch.autograd.grad(embedding.embedding_lookup(table, ids, 3.0).sum(), table)     # a broadcast upstream gradient
    assert ones[1].tolist() == [6.0] * 5 and ones[0].tolist() == [3.0] * 5 and float(ones.sum()) == 4 * 3 * 5


# --- cross-entropy -----------------------------------------------------------------------------------------------------
def exact_xent(logits, labels, weight):
    z = logits.double()
    lse = torch.logsumexp(z, 1)
    ok = (labels >= 0) & (labels < z.shape[1])
    at = torch.where(ok, labels.long(), 0)
    loss = torch.where(ok, lse - z.gather(1, at[:, None])[:, 0], 0.0)
    p = torch.exp(z - lse[:, None])
    onehot = torch.zeros_like(p).scatter_(1, at[:, None], 1.0)
    dz = torch.where(ok[:, None], weight[:, None] * (p - onehot), 0.0)
    return loss, dz, p


def check_xent(logits, labels, weight, loss, dz):
    want, dwant, p = exact_xent(logits, labels, weight)
    z = logits.double()
    spread = (z - z.amax(1, keepdim=True)).abs()
    # what one exponential, relative to its size, and a row's sum can be off by (400: additions of a thread and the exchange)
    e_exp = U * (4 + 3 * spread.clamp(max=60))          # (below e^-60 the term itself is nothing next to the others)
    e_sum = (p * e_exp).sum(1) + 400 * U
    at = labels.clamp(0, logits.shape[1] - 1).long()[:, None]
    tol = e_sum * 1.01 + 2 * U * (spread.gather(1, at)[:, 0] + want.abs() + 20)
    assert bool(((loss.double() - want).abs() <= tol).all())
    if dz is not None:
        tol = weight.abs()[:, None] * (p * (e_exp + e_sum[:, None] + 4 * U) + 2 * U) + half_step(dz.dtype, dwant)
        assert bool(((dz.double() - dwant).abs() <= tol).all())


# classes around one pack, a wave's packs, each step of threads and packs per row, and rows that are streamed
CLASSES = [1, 2, 7, 8, 9, 63, 255, 256, 257, 1000, 1023, 2047, 2049, 4097, 8200, 16385, 32768, 33001, 70000, 131072, 131080, 262147]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", CLASSES)
def test_xent_step_against_64_bits(dtype, classes):
    for tokens in (1, 6):
        g = gen(classes)
        logits = (3 * torch.randn(tokens, classes, device="cuda", generator=g)).to(dtype)
        labels = torch.randint(0, classes, (tokens,), device="cuda", generator=g)
        if tokens > 2:
            labels[1], labels[2] = -1, classes - 1
        dz = torch.full_like(logits, 7.0)
        loss = xent.sparse_softmax_xent_step(logits, labels, dz=dz, grad_scale=0.25)
        w = torch.full((tokens,), 0.25, device="cuda", dtype=torch.float64)
        check_xent(logits, labels, w, loss, dz)
        if tokens > 2:
            assert float(loss[1]) == 0 and bool((dz[1] == 0).all())
        assert torch.equal(xent.sparse_softmax_xent_step(logits, labels.int()), loss)
        inplace = logits.clone()
        assert torch.equal(xent.sparse_softmax_xent_step(inplace, labels, dz=inplace, grad_scale=0.25), loss)
        assert torch.equal(inplace, dz)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", [5, 1000, 9001, 40003, 140000])
def test_xent_strides_and_what_lies_around(dtype, classes):
    room = (2 * torch.randn(5, classes + 11, device="cuda", generator=gen(20))).to(dtype)
    logits = room[1:4, 3:classes + 3]
    for shift in (3, 4):                                 # the same alignment as the logits', and another
        zroom = torch.full((5, classes + 11), 5.0, device="cuda").to(dtype)
        dz = zroom[1:4, shift:classes + shift]
        labels = torch.tensor([0, classes - 1, -5], device="cuda")
        loss = xent.sparse_softmax_xent_step(logits, labels, dz=dz)
        check_xent(logits, labels, torch.ones(3, device="cuda", dtype=torch.float64), loss, dz)
        zroom[1:4, shift:classes + shift] = 5.0
        assert bool((zroom == 5).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", [1, 10, 1025, 5003, 66000])
def test_xent_backward_with_row_gradients(dtype, classes):
    logits = (2 * torch.randn(37, classes, device="cuda", generator=gen(21))).to(dtype).requires_grad_(True)
    labels = torch.randint(-1, classes, (37,), device="cuda", generator=gen(22))
    up = torch.randn(37, device="cuda", generator=gen(23))
    loss = xent.sparse_softmax_xent(logits, labels)
    (dz,) = torch.autograd.grad(loss, logits, up, retain_graph=True)
    check_xent(logits.detach(), labels, up.double(), loss.detach(), dz)
    (mean,) = torch.autograd.grad(loss.mean(), logits)                       # an expanded upstream gradient (stride 0)
    check_xent(logits.detach(), labels, torch.full((37,), 1 / 37, device="cuda", dtype=torch.float64), loss.detach(), mean)


@pytest.mark.parametrize("classes", [6, 700, 9000, 140000])
def test_xent_masks_infinities_and_labels_that_are_no_class(classes):
    z = torch.randn(8, classes, device="cuda", generator=gen(24))
    labels = torch.zeros(8, dtype=torch.long, device="cuda")
    low = torch.finfo(torch.float32).min
    z[0, 1:] = -float("inf")                 # one class left: loss 0
    z[1, :] = -float("inf")                  # none left
    z[2, 3] = float("nan")
    z[3, 4] = float("inf")
    z[4, 1::2] = -float("inf")               # every other class masked
    z[5, 1:] = low                           # masked by the lowest value
    labels[6], labels[7] = classes, -3
    z[7] = float("nan")                      # padding is not looked at
    loss = xent.sparse_softmax_xent_step(z, labels)
    dz = torch.empty_like(z)
    assert torch.equal(torch.nan_to_num(loss, 99.0), torch.nan_to_num(xent.sparse_softmax_xent_step(z, labels, dz=dz), 99.0))
    assert float(loss[0]) == 0 and bool((dz[0] == 0).all())
    assert all(math.isnan(float(loss[r])) and bool(dz[r].isnan().any()) for r in (1, 2, 3, 6))
    assert bool(dz[6].isnan().all())
    assert float(loss[5]) == 0 and bool((dz[5] == 0).all())
    assert float(loss[7]) == 0 and bool((dz[7] == 0).all())
    rest = torch.tensor([0, 4], device="cuda")
    check_xent(z[rest], labels[rest], torch.ones(2, device="cuda", dtype=torch.float64), loss[rest], dz[rest])
    assert bool((dz[4, 1::2] == 0).all())
    logits = z.clone().requires_grad_(True)
    rows = xent.sparse_softmax_xent(logits, labels)
    (g,) = torch.autograd.grad(rows, logits, torch.ones_like(rows))
    assert torch.equal(torch.nan_to_num(rows.detach(), 99.0), torch.nan_to_num(loss, 99.0))
    assert torch.equal(g.isnan().any(1), dz.isnan().any(1)) and bool((g[7] == 0).all()) and bool((g[0] == 0).all())


def test_xent_many_rows_equal_one_by_one():
    logits = (2 * torch.randn(300, 2000, device="cuda", generator=gen(25))).bfloat16()
    labels = torch.randint(-1, 2000, (300,), device="cuda", generator=gen(26))
    loss = xent.sparse_softmax_xent_step(logits, labels)
    for t in (0, 1, 77, 299):
        assert torch.equal(xent.sparse_softmax_xent_step(logits[t:t + 1], labels[t:t + 1]), loss[t:t + 1])
    assert xent.sparse_softmax_xent_step(logits[:0], labels[:0]).shape == (0,)


# --- streams, graphs, devices ----------------------------------------------------------------------------------------------
def test_operators_on_a_side_stream_and_in_a_replayed_graph():
    rows, dim, tokens = 300, 96, 5000
    table = torch.randn(rows, dim, device="cuda", generator=gen(30))
    ids = make_ids(tokens, rows, 31)
    g = torch.randn(tokens, dim, device="cuda", generator=gen(32))
    logits = torch.randn(50, 999, device="cuda", generator=gen(33))
    labels = torch.randint(-1, 999, (50,), device="cuda", generator=gen(34))
    lr = torch.full((1,), 0.125, device="cuda")
    updated = table.clone()

    def step():
        dz = torch.empty_like(logits)
        return (embedding.lookup(table, ids, 2.0), embedding.lookup_grad(ids, g, rows, 2.0),
                xent.sparse_softmax_xent_step(logits, labels, dz=dz), dz, embedding.lookup_sgd(updated, ids, g, lr))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for k in range(3):
        ids.copy_(make_ids(tokens, rows, 40 + k))
        g.copy_(torch.randn(tokens, dim, device="cuda", generator=gen(50 + k)))
        logits.copy_(torch.randn(50, 999, device="cuda", generator=gen(60 + k)))
        updated.copy_(table)
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        updated.copy_(table)
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals_of_gpu_operands():
    table = torch.zeros(4, 8, device="cuda")
    ids = torch.zeros(3, dtype=torch.long, device="cuda")
    g = torch.zeros(3, 8, device="cuda")
    lr = torch.zeros(1, device="cuda")
    bad = [lambda: embedding.lookup(table.double(), ids), lambda: embedding.lookup(table, ids.float()),
           lambda: embedding.lookup(table, ids.cpu()), lambda: embedding.lookup(table.t(), ids),
           lambda: embedding.lookup(table[0], ids), lambda: embedding.lookup(table, ids, out=table[:3]),
           lambda: embedding.lookup(table, ids, out=torch.zeros(3, 7, device="cuda")),
           lambda: embedding.lookup(table[:0], ids), lambda: embedding.lookup(table[:, :0], ids),
           lambda: embedding.lookup_grad(ids, g[:2], 4), lambda: embedding.lookup_grad(ids, g, 0),
           lambda: embedding.lookup_grad(ids, g.double(), 4), lambda: embedding.lookup_grad(ids, table[:3], 4, out=table),
           lambda: embedding.lookup_sgd(table, ids, g.half(), lr), lambda: embedding.lookup_sgd(table, ids, g[:, :7], lr),
           lambda: embedding.lookup_sgd(table, ids, g, lr.double()), lambda: embedding.lookup_sgd(table, ids, table[:3], lr),
           lambda: embedding.lookup_sgd(table, ids, g, torch.zeros(2, device="cuda")),
           lambda: xent.sparse_softmax_xent_step(table, ids), lambda: xent.sparse_softmax_xent_step(table[:3], ids.float()),
           lambda: xent.sparse_softmax_xent_step(table[:3], ids, dz=torch.zeros(3, 7, device="cuda")),
           lambda: xent.sparse_softmax_xent_step(table[:3], ids, dz=table[1:4]),
           lambda: xent.sparse_softmax_xent_step(table[:3].double(), ids),
           lambda: xent.sparse_softmax_xent_step(table[:3], ids.view(3, 1)),
           lambda: xent.sparse_softmax_xent_step(table[:3, :0], ids)]
    for k, call in enumerate(bad):
        with pytest.raises(hb.HipKernelError):
            call()
            pytest.fail(f"call {k} was not refused")


def test_forward_and_backward_in_a_replayed_graph():
    """Fresh leaves inside the capture, so that no eager graph of them lives next to it.  (The rows of the table are the logits.)"""
    rows, classes, tokens = 700, 333, 4500
    table = torch.randn(rows, classes, device="cuda", generator=gen(70))
    ids = make_ids(tokens, rows, 71)
    labels = torch.randint(-1, classes, (tokens,), device="cuda", generator=gen(73))

    def step():
        leaf = table.detach().requires_grad_(True)
        losses = xent.sparse_softmax_xent(embedding.embedding_lookup(leaf, ids, 2.0), labels)
        return (losses.detach(), *torch.autograd.grad(losses, leaf, torch.full_like(losses, 0.25)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for k in range(3):
        ids.copy_(make_ids(tokens, rows, 80 + k))
        labels.copy_(torch.randint(-1, classes, (tokens,), device="cuda", generator=gen(90 + k)))
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_calls_on_two_streams_at_once():
    """Workspaces belong to a call: two row updates and gradients side by side do what they do one after the other."""
    rows, dim, tokens = 2000, 128, 20000
    args = [(make_ids(tokens, rows, 100 + k), torch.randn(tokens, dim, device="cuda", generator=gen(110 + k))) for k in range(2)]
    want = [embedding.lookup_grad(i, g, rows) for i, g in args]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(10):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(embedding.lookup_grad(*args[k], rows))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(x, want[k]) for x in got[k])


def test_no_second_derivatives():
    """The backward passes are launches, not graphs: a second derivative is refused, not silently left out."""
    table = torch.randn(5, 4, device="cuda", generator=gen(120)).requires_grad_(True)
    ids = torch.tensor([0, 1, 1], device="cuda")
    for losses in (embedding.embedding_lookup(table, ids).square().sum(1), xent.sparse_softmax_xent(table[:3] * 2, ids)):
        (g,) = torch.autograd.grad(losses.sum(), table, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), table)


@pytest.mark.parametrize("gap", [0, 4])
@pytest.mark.parametrize("rows", [300, 60000])
def test_gradient_of_a_table_over_what_was_there(rows, gap):
    """Rows that do not occur become zeros whoever clears them (60000 x 1024 is more than the sort's launches take), the
    elements between the rows stay as they were."""
    dim, tokens = 1024, 4100
    ids = make_ids(tokens, rows, 130, kind="uniform")
    g = torch.randn(tokens, dim, device="cuda", generator=gen(131))
    room = torch.full((rows, dim + gap), float("nan"), device="cuda")
    embedding.lookup_grad(ids, g, rows, out=room[:, :dim])
    want, size, count = exact_sums(ids, g, rows)
    # (an fp32 sum of n terms is off by less than n 2^-24 of the sum of their magnitudes)
    assert bool(((room[:, :dim].double() - want).abs() <= count[:, None] * 2.0 ** -24 * size).all())
    assert bool(room[:, dim:].isnan().all()) and (rows == 300 or bool((count == 0).any()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", [66000, 131080, 262147])
def test_xent_of_many_long_rows(dtype, classes):
    """65 rows: one block each (64 would be cut into slices)."""
    logits = (3 * torch.randn(65, classes, device="cuda", generator=gen(140))).to(dtype)
    labels = torch.randint(0, classes, (65,), device="cuda", generator=gen(141))
    labels[1] = -1
    dz = torch.empty_like(logits)
    loss = xent.sparse_softmax_xent_step(logits, labels, dz=dz, grad_scale=0.5)
    for rows in (slice(0, 9), slice(56, 65)):            # (64-bit copies of all of them would take gigabytes)
        n = rows.stop - rows.start
        check_xent(logits[rows], labels[rows], torch.full((n,), 0.5, device="cuda", dtype=torch.float64), loss[rows], dz[rows])
    inplace = logits.clone()
    assert torch.equal(xent.sparse_softmax_xent_step(inplace, labels, dz=inplace, grad_scale=0.5), loss) and torch.equal(inplace, dz)


@pytest.mark.parametrize("shift", [0, 1, 3])
@pytest.mark.parametrize("dtype", TYPES)
def test_xent_of_rows_in_slices_labels_at_their_ends(dtype, shift):
    """Slices are 1024 packs of 16 bytes of memory: labels on either side of their borders, in a row that starts inside a pack."""
    per_slice = 1024 * 16 // dtype.itemsize
    classes = 20 * per_slice + 5
    at = [0, classes - 1, classes - 5] + [k * per_slice - shift + d for k in (1, 7, 20) for d in (-1, 0, 1)]
    room = (2 * torch.randn(classes + shift, device="cuda", generator=gen(142))).to(dtype)
    logits = room[shift:].unsqueeze(0)
    for label in at:
        labels = torch.tensor([label], device="cuda")
        dz = torch.empty_like(logits)
        loss = xent.sparse_softmax_xent_step(logits, labels, dz=dz)
        check_xent(logits, labels, torch.ones(1, device="cuda", dtype=torch.float64), loss, dz)
        assert torch.equal(xent.sparse_softmax_xent_step(logits, labels), loss)
        inplace = room.clone()[shift:].unsqueeze(0)
        assert torch.equal(xent.sparse_softmax_xent_step(inplace, labels, dz=inplace), loss) and torch.equal(inplace, dz)
