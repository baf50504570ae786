"""Several train ops in one session: a step of one leaves alone what the others train.  (CPU sessions here, the same on a GPU with
``-m gpu``.)"""
import numpy as np
import pytest
import torch

import distributed_tensorflow_amd as tf


def stack(widths, batch=16):
    """A graph that the engines recognise: placeholders, variables, loss and a feed for them."""
    rng = np.random.RandomState(5)
    x, y = tf.placeholder(tf.float32, [None, widths[0]]), tf.placeholder(tf.float32, [None, widths[-1]])
    w = [tf.Variable(tf.random_normal([a, b], stddev=a ** -0.5), name=f"w{k}") for k, (a, b) in enumerate(zip(widths, widths[1:]))]
    b = [tf.Variable(tf.zeros([m]), name=f"b{k}") for k, m in enumerate(widths[1:])]
    h = x
    for k in range(len(w)):
        h = tf.add(tf.matmul(h, w[k]), b[k])
        h = tf.nn.relu(h) if k + 1 < len(w) else h
    loss = tf.reduce_mean(tf.nn.softmax_cross_entropy_with_logits(labels=y, logits=h))
    feed = {x: rng.rand(batch, widths[0]).astype(np.float32),
            y: np.eye(widths[-1], dtype=np.float32)[rng.randint(0, widths[-1], batch)]}
    return w, b, loss, feed


def _engine_step_beside_another_op(make, widths):
    """An engine's gradient pass writes its own slices of the gradient slab: what an earlier step of another op left next to them
    must not be applied again."""
    with tf.Graph().as_default():
        w, b, loss, feed = stack(widths)
        other = tf.Variable(tf.zeros([5, 3]), name="other")
        pull = tf.reduce_sum(tf.square(tf.subtract(other, tf.constant(np.ones((5, 3), np.float32)))))
        step = tf.train.get_or_create_global_step()
        aside = tf.train.GradientDescentOptimizer(0.1).minimize(pull, var_list=[other])
        train = make().minimize(loss, global_step=step, var_list=w + b)
        with tf.Session() as sess:
            sess.run(tf.global_variables_initializer())
            for k in range(3):
                sess.run(aside)
                kept = sess.var_tensor(other).clone()
                before = [sess.var_tensor(v).clone() for v in w + b]
                sess.run(train, feed_dict=feed)
                sess.run([train, loss], feed_dict=feed)
                assert torch.equal(sess.var_tensor(other), kept), k
                assert not any(torch.equal(sess.var_tensor(v), p) for v, p in zip(w + b, before))
                assert sess.run(step) == 2 * (k + 1)
            # 1 - (1 - 2 * 0.1)^3 of the way, in three fp32 steps
            assert float((sess.var_tensor(other).cpu().double() - (1 - 0.8 ** 3)).abs().max()) < 1e-6
            assert sess.fused_steps == 6


MAKERS = {"muon": lambda: tf.train.MuonOptimizer(0.1, sgd_learning_rate=0.3), "sgd": lambda: tf.train.GradientDescentOptimizer(0.3)}


@pytest.mark.parametrize("kind", sorted(MAKERS))
@pytest.mark.parametrize("widths", [(20, 30, 6), (20, 30, 24, 6)])
def test_engine_step_beside_another_op_on_the_cpu(kind, widths):
    with tf.device("/cpu:0"):
        _engine_step_beside_another_op(MAKERS[kind], widths)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", sorted(MAKERS))
@pytest.mark.parametrize("widths", [(20, 30, 6), (20, 30, 24, 6)])
def test_engine_step_beside_another_op_on_the_gpu(kind, widths):
    _engine_step_beside_another_op(MAKERS[kind], widths)


@pytest.mark.parametrize("resident", [False, True])
@pytest.mark.parametrize("widths", [(20, 30, 6), (20, 30, 24, 6)])
def test_engine_step_beside_another_op_on_a_parameter_server(widths, resident):
    """The same over TCP, where every step pushes the gradient slab: through ``sess.run``, and by the device-resident trainers."""
    from cluster_utils import cluster_dict

    from distributed_tensorflow_amd.data import DeviceDataset
    from distributed_tensorflow_amd.parallel.dense_trainer import PsDenseResidentTrainer
    from distributed_tensorflow_amd.parallel.ps_resident import PsResidentTrainer

    cluster = tf.train.ClusterSpec(cluster_dict(1, 1))
    cfg = tf.ConfigProto(allow_soft_placement=True, operation_timeout_in_ms=20000)
    ps, worker = tf.train.Server(cluster, "ps", 0, config=cfg), tf.train.Server(cluster, "worker", 0, config=cfg)
    try:
        g = tf.Graph()
        with g.as_default(), tf.device(tf.train.replica_device_setter(worker_device="/job:worker/task:0/cpu:0", cluster=cluster)):
            w, b, loss, feed = stack(widths)
            other = tf.Variable(tf.zeros([5, 3]), name="other")
            pull = tf.reduce_sum(tf.square(tf.subtract(other, tf.constant(np.ones((5, 3), np.float32)))))
            step = tf.train.get_or_create_global_step()
            aside = tf.train.GradientDescentOptimizer(0.1).minimize(pull, var_list=[other])
            train = tf.train.GradientDescentOptimizer(0.3).minimize(loss, global_step=step, var_list=w + b)
            init = tf.global_variables_initializer()
        sv = tf.train.Supervisor(graph=g, is_chief=True, global_step=step, init_op=init)
        sess = sv.prepare_or_wait_for_session(worker.target)
        sess.run(aside)
        kept, before = sess.run(other), sess.run(w[0])
        if resident:
            ds = DeviceDataset(*feed.values(), sess.device, 8, seed=3)
            trainer = (PsResidentTrainer if len(widths) == 3 else PsDenseResidentTrainer)(sess, train, ds, 8)
            trainer.run_steps(2)
        else:
            sess.run(train, feed_dict=feed)
            sess.run([train, loss], feed_dict=feed)
        assert np.array_equal(sess.run(other), kept)
        after = sess.run(w[0])
        assert not np.array_equal(after, before)
        sess.run(aside)
        assert np.array_equal(sess.run(w[0]), after) and abs(float(sess.run(other)[0, 0]) - 0.36) < 1e-6
        assert sess.run(step) == 2
        kept = sess.run(other)
        if resident:
            trainer.run_steps(1)
        else:
            sess.run(train, feed_dict=feed)
        assert np.array_equal(sess.run(other), kept) and not np.array_equal(sess.run(w[0]), after)
        assert sess.run(step) == 3
        sv.stop()
        sess.close()
    finally:
        worker.stop()
        ps.stop()


def test_resident_trainers_refuse_muon():
    """Their steps are plain gradient descent: a MuonOptimizer op must not be trained with it instead."""
    from cluster_utils import cluster_dict

    from distributed_tensorflow_amd.data import DeviceDataset
    from distributed_tensorflow_amd.parallel.dense_trainer import DenseResidentTrainer, PsDenseResidentTrainer
    from distributed_tensorflow_amd.parallel.ps_resident import PsResidentTrainer

    for widths in ((20, 30, 6), (20, 30, 24, 6)):
        with tf.Graph().as_default(), tf.device("/cpu:0"):
            w, b, loss, feed = stack(widths)
            train = tf.train.MuonOptimizer(0.1).minimize(loss, global_step=tf.train.get_or_create_global_step())
            with tf.Session() as sess:
                sess.run(tf.global_variables_initializer())
                ds = DeviceDataset(*feed.values(), sess.device, 8, seed=3)
                start = sess.theta.clone()
                for trainer in (DenseResidentTrainer, PsDenseResidentTrainer, PsResidentTrainer):
                    with pytest.raises(NotImplementedError):
                        trainer(sess, train, ds, 8)
                assert torch.equal(sess.theta, start)
    cluster = tf.train.ClusterSpec(cluster_dict(1, 1))
    cfg = tf.ConfigProto(allow_soft_placement=True, operation_timeout_in_ms=20000)
    ps, worker = tf.train.Server(cluster, "ps", 0, config=cfg), tf.train.Server(cluster, "worker", 0, config=cfg)
    try:
        g = tf.Graph()
        with g.as_default(), tf.device(tf.train.replica_device_setter(worker_device="/job:worker/task:0/cpu:0", cluster=cluster)):
            w, b, loss, feed = stack((20, 30, 24, 6))
            step = tf.train.get_or_create_global_step()
            train = tf.train.MuonOptimizer(0.1).minimize(loss, global_step=step)
            init = tf.global_variables_initializer()
        sv = tf.train.Supervisor(graph=g, is_chief=True, global_step=step, init_op=init)
        sess = sv.prepare_or_wait_for_session(worker.target)
        with pytest.raises(NotImplementedError):
            PsDenseResidentTrainer(sess, train, DeviceDataset(*feed.values(), sess.device, 8, seed=3), 8)
        assert sess.run(step) == 0
        sv.stop()
        sess.close()
    finally:
        worker.stop()
        ps.stop()


def _gradient_of_a_table_inside_a_loss():
    """A loss that holds the gradient of another one: while the train op looks rows up as leaves, that gradient is still the
    table's."""
    with tf.Graph().as_default():
        ids = tf.placeholder(tf.int64, [None])
        table = tf.Variable(tf.random_normal([5, 3]), name="table")
        inner = tf.reduce_sum(tf.square(tf.nn.embedding_lookup(table, ids)))
        opt = tf.train.GradientDescentOptimizer(0.1)
        (g, _), = opt.compute_gradients(inner, [table])
        loss = tf.add(tf.reduce_sum(tf.nn.embedding_lookup(table, ids)), tf.reduce_sum(tf.square(g)))
        train = opt.minimize(loss)
        with tf.Session() as sess:
            sess.run(tf.global_variables_initializer())
            start = sess.var_tensor(table).cpu().double().clone()
            count = torch.tensor([0.0, 2.0, 0.0, 1.0, 0.0]).double()[:, None]
            want = float((count * start).sum() + (2 * count * start).square().sum())
            feed = {ids: np.array([1, 3, 1])}
            assert abs(sess.run(loss, feed_dict=feed) - want) < 1e-5 * abs(want) + 1e-5
            _, got = sess.run([train, loss], feed_dict=feed)
            assert abs(got - want) < 1e-5 * abs(want) + 1e-5
            # (a gradient is a constant of the step: the sum of the rows alone moves them)
            assert float((sess.var_tensor(table).cpu().double() - (start - 0.1 * count)).abs().max()) < 1e-6


def test_gradient_of_a_table_inside_a_loss_on_the_cpu():
    with tf.device("/cpu:0"):
        _gradient_of_a_table_inside_a_loss()


@pytest.mark.gpu
def test_gradient_of_a_table_inside_a_loss_on_the_gpu():
    _gradient_of_a_table_inside_a_loss()


def _muon_leaves_alone_what_its_loss_does_not_read(with_table):
    """A matrix in the var_list of a train op whose loss does not depend on it has no gradient: neither it nor its momentum moves,
    also when another op has left that momentum behind."""
    with tf.Graph().as_default():
        ids = tf.placeholder(tf.int64, [None])
        x = tf.constant(np.random.RandomState(1).rand(7, 8).astype(np.float32))
        read = tf.nn.embedding_lookup(tf.Variable(tf.random_normal([9, 8]), name="table"), ids) if with_table else x
        w = [tf.Variable(tf.random_normal([8, 5]), name=f"w{k}") for k in range(2)]
        losses = [tf.reduce_mean(tf.square(tf.matmul(r, v))) for r, v in zip((x, read), w)]
        opt = tf.train.MuonOptimizer(0.1)
        first = opt.minimize(losses[0], var_list=w[:1])
        both = opt.minimize(losses[1])                  # every trainable variable, w[0] among them
        with tf.Session() as sess:
            sess.run(tf.global_variables_initializer())
            sess.run(first)
            slot = next(v for v in tf.global_variables() if v.op_name == "w0/Muon")
            start = [sess.var_tensor(v).clone() for v in (w[0], slot, w[1])]
            assert float(start[1].abs().max()) > 0
            for _ in range(2):
                sess.run(both, feed_dict={ids: np.array([1, 2, 2])})
            now = [sess.var_tensor(v) for v in (w[0], slot, w[1])]
            assert torch.equal(now[0], start[0]) and torch.equal(now[1], start[1]) and not torch.equal(now[2], start[2])
            sess.run(first)
            assert not torch.equal(sess.var_tensor(w[0]), start[0])


@pytest.mark.parametrize("with_table", [False, True])
def test_muon_leaves_alone_what_its_loss_does_not_read_on_the_cpu(with_table):
    with tf.device("/cpu:0"):
        _muon_leaves_alone_what_its_loss_does_not_read(with_table)


@pytest.mark.gpu
@pytest.mark.parametrize("with_table", [False, True])
def test_muon_leaves_alone_what_its_loss_does_not_read_on_the_gpu(with_table):
    _muon_leaves_alone_what_its_loss_does_not_read(with_table)


def test_a_fetched_variable_stays_as_it_was_fetched():
    """A CPU session's variables lie in host memory: what ``sess.run`` hands out is a copy of it."""
    with tf.Graph().as_default(), tf.device("/cpu:0"):
        ids = tf.placeholder(tf.int64, [None])
        table = tf.Variable(tf.ones([4, 3]), name="table")
        train = tf.train.GradientDescentOptimizer(0.5).minimize(tf.reduce_sum(tf.nn.embedding_lookup(table, ids)))
        with tf.Session() as sess:
            sess.run(tf.global_variables_initializer())
            fetched, same = sess.run(table), sess.run(tf.identity(table))
            sess.run(train, feed_dict={ids: np.array([2])})
            assert (fetched == 1).all() and (same == 1).all()
            assert (sess.run(table)[2] == 0.5).all()
            fetched[:] = 7
            assert (sess.run(table)[0] == 1).all()
