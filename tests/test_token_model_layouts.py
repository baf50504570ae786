"""Operands of the differentiable token-model operators whose rows do not lie in memory one behind the other: a transposed table
(input and output embedding shared), tables and logits expanded from one row.  (CPU tensors here, the same on a GPU with
``-m gpu``.)

Tolerance: values are of size one and every result is a sum of at most 40 fp32 products or exponentials, 40 * 2^-24 = 2.4e-6 of
sums of magnitudes below 8; results are compared within 4e-5."""
import numpy as np
import pytest
import torch

import distributed_tensorflow_amd as tf
from distributed_tensorflow_amd.ops import embedding, xent

HIDDEN, V = 12, 40


def _shared_embedding_in_a_graph():
    """logits = scale * W^T[ids] W: the lookup reads the transposed output matrix."""
    with tf.Graph().as_default():
        ids, labels = tf.placeholder(tf.int64, [None]), tf.placeholder(tf.int64, [None])
        w = tf.Variable(tf.random_normal([HIDDEN, V], stddev=0.5), name="w")
        logits = tf.matmul(tf.nn.embedding_lookup(tf.transpose(w), ids, scale=1.5), w)
        loss = tf.reduce_mean(tf.nn.sparse_softmax_cross_entropy_with_logits(labels=labels, logits=logits))
        train = tf.train.GradientDescentOptimizer(0.5).minimize(loss)
        i, lab = np.array([1, 1, 39, 0, -1, V, 7]), np.array([2, 3, 3, 0, 5, 6, -1])
        with tf.Session() as sess:
            sess.run(tf.global_variables_initializer())
            p = sess.var_tensor(w).cpu().double().requires_grad_(True)
            inside = torch.tensor((i >= 0) & (i < V))
            x = 1.5 * p.t()[torch.tensor(i).clamp(0, V - 1)] * inside[:, None]
            logp = torch.log_softmax(x @ p, 1)
            want = -(logp[torch.arange(7), torch.tensor(lab).clamp(min=0)] * torch.tensor(lab >= 0)).sum() / 7
            (g,) = torch.autograd.grad(want, p)
            _, got = sess.run([train, loss], feed_dict={ids: i, labels: lab})
            assert abs(got - float(want.detach())) < 4e-5
            assert float((sess.var_tensor(w).cpu().double() - (p.detach() - 0.5 * g)).abs().max()) < 4e-5


def _expanded_operands(device):
    g = torch.Generator().manual_seed(3)
    ids, labels = torch.tensor([3, 0, 3, -1]).to(device), torch.tensor([4, 1, -1, 0]).to(device)
    up = torch.randn(4, V, generator=g).to(device)
    row = torch.randn(V, generator=g).to(device).requires_grad_(True)
    out = embedding.embedding_lookup(row.expand(5, V), ids, 0.5)
    (got,) = torch.autograd.grad(out, row, up)
    inside = torch.tensor([1, 1, 1, 0])[:, None]
    assert float((out.detach().cpu().double() - 0.5 * row.detach().cpu().double() * inside).abs().max()) < 4e-5
    assert float((got.cpu().double() - 0.5 * (up.cpu().double() * inside).sum(0)).abs().max()) < 4e-5
    for shape in ((1, V), (4, 1)):
        base = torch.randn(shape, generator=g).to(device).requires_grad_(True)
        loss = xent.sparse_softmax_xent(base.expand(4, V), labels)
        (got,) = torch.autograd.grad(loss.sum(), base)
        q = base.detach().cpu().double().requires_grad_(True)
        logp = torch.log_softmax(q.expand(4, V), 1)
        want = -logp[torch.arange(4), labels.cpu().clamp(min=0)] * (labels.cpu() >= 0)
        (g64,) = torch.autograd.grad(want.sum(), q)
        assert float((loss.detach().cpu().double() - want.detach()).abs().max()) < 4e-5
        assert float((got.cpu().double() - g64).abs().max()) < 4e-5


def _transposed_operands(device):
    g = torch.Generator().manual_seed(4)
    w = torch.randn(HIDDEN, V, generator=g).to(device).requires_grad_(True)
    ids = torch.tensor([[3, 0], [39, -1]], dtype=torch.int32).to(device)
    up = torch.randn(2, 2, HIDDEN, generator=g).to(device)
    out = embedding.embedding_lookup(w.t(), ids, 2.0)
    (got,) = torch.autograd.grad(out, w, up)
    want = torch.zeros(V, HIDDEN, dtype=torch.float64)
    for k, v in enumerate(ids.cpu().reshape(-1).tolist()):
        if v >= 0:
            assert float((out.detach().cpu().reshape(4, -1)[k].double() - 2.0 * w.detach().cpu()[:, v].double()).abs().max()) < 4e-5
            want[v] += 2.0 * up.cpu().reshape(4, -1)[k].double()
    assert float((got.cpu().double() - want.t()).abs().max()) < 4e-5


def test_shared_embedding_in_a_graph_on_the_cpu():
    with tf.device("/cpu:0"):
        _shared_embedding_in_a_graph()


@pytest.mark.parametrize("check", [_expanded_operands, _transposed_operands])
def test_operands_on_the_cpu(check):
    check(torch.device("cpu"))


@pytest.mark.gpu
def test_shared_embedding_in_a_graph_on_the_gpu():
    _shared_embedding_in_a_graph()


@pytest.mark.gpu
@pytest.mark.parametrize("check", [_expanded_operands, _transposed_operands])
def test_operands_on_the_gpu(check):
    check(torch.device("cuda"))
