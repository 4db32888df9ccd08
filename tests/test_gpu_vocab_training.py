"""The vocabulary operators and the optimizers as a distillation step uses them, each stage feeding the
next on the GPU, against the same steps in float64."""
import numpy as np
import pytest
import torch

from oracle import lans_f64, sgd_f32, vocab_f64
from oracle.lans_f64 import LansHParams

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24


def _targets(n, vocab, k, seed):
    rng = np.random.default_rng([seed, n, vocab, k])
    idx = np.stack([rng.permutation(vocab)[:k] for _ in range(n)])
    idx[rng.random((n, k)) < 0.1] = -1
    labels = rng.integers(0, vocab, n)
    pad = rng.random(n) < 0.2  # a padded batch: neither target nor token
    idx[pad], labels[pad] = -1, -100
    ids = np.minimum(np.exp(rng.uniform(0, np.log(vocab), n)).astype(np.int64), vocab - 1)
    ids[pad] = -1
    t = rng.normal(3, 2, (n, k)).astype(np.float32)
    return ids, idx, t, labels


def _distill_bound(r, vocab, spread, z_off, temperature, soft, hard, dl):
    """Bound on the gradient's error for logits off by z_off (a column): their softmax changes by at most the
    factor exp(2 z_off / T), and the kernel's own error is 2^-24 times the roundings of an exponential of
    `spread` and of a sum of `vocab` terms."""
    own = U * (300 + 8 * (spread + np.log2(vocab)))
    return (r["soft"] * (own + 2.2 * z_off / temperature) + r["p"] * own + r["hard"] * (own + 2.2 * z_off)
            + 2 * U * np.abs(r["dlogits"]) + 2.0 ** -126)


@pytest.mark.parametrize("shape", [(3, 37), (700,)])
def test_tied_table(native_libs, shape):
    """Token table and output projection are one tensor: its gradient is the projection's plus the lookup's,
    accumulated in place, and feeds the optimizer."""
    from raf_amd import op

    n, vocab, width, k = int(np.prod(shape)), 1003, 48, 11
    temperature, soft, hard, scale = 2.0, 0.7, 0.3, float(np.float32(np.sqrt(width)))
    ids, idx, t, labels = _targets(n, vocab, k, 1)
    rng = np.random.default_rng(2)
    table = rng.normal(0, 0.1, (vocab, width)).astype(np.float32)
    dl = np.full(1, 128.0 / n, np.float32)
    dev = lambda x, *s: torch.from_numpy(x).to(DEV).reshape(*s) if s else torch.from_numpy(x).to(DEV)
    w, ids_d = dev(table), dev(ids, *shape)
    more = dict(temperature=temperature, soft_weight=soft, labels=dev(labels, *shape), hard_weight=hard)

    x = op.embedding(w, ids_d, scale=scale)
    logits = x @ w.t()
    loss, dlogits = op.topk_distill_step(logits, dev(idx, *shape, k), dev(t, *shape, k), dev(dl), **more)
    grad = (dlogits.reshape(n, vocab).t() @ x.reshape(n, width)).contiguous()
    dx = dlogits @ w
    assert op.embedding_dx(dx, ids_d, vocab, scale=scale, grad=grad) is grad

    w64 = table.astype(np.float64)
    x64 = vocab_f64.embedding(w64, ids, scale)
    z64 = x64 @ w64.T
    r = vocab_f64.topk_distill(z64, idx, t, temperature, soft, labels, hard, dl)
    # A product of length c is off by (c + 2) 2^-24 times the sum of magnitudes; inputs' errors pass through.
    z_off = ((width + 3) * U * (np.abs(x64) @ np.abs(w64).T)).max(1, keepdims=True)
    spread = (z64.max(1) - z64.min(1))[:, None] * 1.4427
    dz_off = _distill_bound(r, vocab, spread, z_off, temperature, soft, hard, dl)
    dz, dz_size = r["dlogits"], np.abs(r["dlogits"]) + dz_off
    assert (np.abs(dlogits.reshape(n, vocab).double().cpu().numpy() - dz) <= dz_off).all()
    head, head_off = dz.T @ x64, dz_off.T @ np.abs(x64) * 1.01 + (n + 3) * U * (dz_size.T @ np.abs(x64))
    dx64, dx_off = dz @ w64, dz_off @ np.abs(w64) + (vocab + 2) * U * (dz_size @ np.abs(w64))
    token, size, count = vocab_f64.embedding_dx(dx64, ids, vocab, scale)
    _, off, _ = vocab_f64.embedding_dx(dx_off, ids, vocab, scale)
    bound = head_off + off * 1.01 + (count[:, None] + 3) * U * (size + off) + 2 * U * np.abs(head + token)
    got = grad.double().cpu().numpy()
    assert (np.abs(got - (head + token)) <= bound).all()
    absent = np.setdiff1d(np.arange(vocab), ids)
    assert (np.abs(got - head)[absent] <= head_off[absent] + 2 * U * np.abs(head[absent])).all()  # rows without tokens

    # Central differences of the loss in float64 along a direction of the table: what is differentiated is
    # smooth, so their own error is of order eps^2 (a third of what halving eps changes) and the sum's rounding.
    direction = np.random.default_rng(3).normal(0, 1, table.shape)

    def total(e):
        v = w64 + e * direction
        emb = vocab_f64.embedding(v, ids, scale)
        return float(np.sum(vocab_f64.topk_distill(emb @ v.T, idx, t, temperature, soft, labels, hard)["loss"]) * dl[0])

    slopes = [(total(e) - total(-e)) / (2 * e) for e in (2e-5, 1e-5)]
    noise = 1e-12 * abs(total(0.0)) / 1e-5 + abs(slopes[0] - slopes[1])
    assert abs(np.sum(got * direction) - slopes[1]) <= noise + np.sum(bound * np.abs(direction))

    # and the optimizer takes it as it is: a weight is rounded once, its change after fewer than 100 roundings
    # of terms no larger than the largest change.
    hp = LansHParams(learning_rate=0.01)
    g0 = grad.cpu().numpy()
    want = lans_f64.lans_step([g0], [table], [np.zeros_like(table)], [np.zeros_like(table)], 1.0, hp)
    m, v, step = torch.zeros_like(w), torch.zeros_like(w), torch.ones((), device=DEV)
    op.lans([grad, w, m, v], step, hp.learning_rate, hp.beta1, hp.beta2, hp.eps, hp.bias_correction, hp.weight_decay,
            hp.grad_averaging, hp.mode, hp.normalize_grad)
    new = want[0][0].astype(np.float64)
    assert (np.abs(w.double().cpu().numpy() - new) <= 2 * U * np.abs(new) + 100 * U * np.abs(new - table).max()).all()


def test_bigram_model_eager_and_captured(native_libs):
    """A table of logits by the last token: lookup, loss, gradient and update are this library's alone.  Three
    steps, eager and as a captured graph with other work between its replays, agree bit for bit and
    each follows float64 from the state before it."""
    from raf_amd import op

    n, vocab, k, lr, mu = 900, 257, 5, 0.05, 0.9
    rng = np.random.default_rng(4)
    start = rng.normal(0, 1, (vocab, vocab)).astype(np.float32)
    batches = [_targets(n, vocab, k, 10 + s) for s in range(3)]
    more = dict(temperature=1.5, hard_weight=0.5)

    def step(table, v, ids, idx, t, labels, dl):
        logits = op.embedding(table, ids)
        loss, dlogits = op.topk_distill_step(logits, idx, t, dl, labels=labels, **more)
        loss2, stats = op.topk_distill(logits, idx, t, labels=labels, **more)
        again = op.topk_distill_dx(dl, logits, idx, t, stats, labels=labels, **more)
        grad = op.embedding_dx(dlogits, ids, vocab)
        v1, x1 = op.sgd(table, grad, v, lr, mu)
        return loss, dlogits, loss2, again, grad, v1, x1

    dev = [tuple(torch.from_numpy(x).to(DEV) for x in b) for b in batches]
    dl = torch.full((1,), 1.0 / n, device=DEV)
    inputs = [torch.from_numpy(start).to(DEV), torch.zeros(vocab, vocab, device=DEV), *[x.clone() for x in dev[0]], dl]
    step(*inputs)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured = step(*inputs)
    table, v = inputs[0].clone(), inputs[1].clone()
    for s in range(3):
        eager = step(table, v, *dev[s], dl)
        for to, x in zip(inputs, (table, v, *dev[s])):
            to.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, eager)), s
        loss, dlogits, loss2, again, grad, v1, x1 = eager

        ids, idx, t, labels = batches[s]
        z = vocab_f64.embedding(table.cpu().numpy(), ids)
        r = vocab_f64.topk_distill(z, idx, t, 1.5, 1.0, labels, 0.5, dl.cpu().numpy())
        spread = (z.max(1) - z.min(1))[:, None] * 1.4427
        off = _distill_bound(r, vocab, spread, 0.0, 1.5, 1.0, 0.5, None)
        for g in (dlogits, again):
            assert (np.abs(g.double().cpu().numpy() - r["dlogits"]) <= off).all()
        sums, size, count = vocab_f64.embedding_dx(dlogits.cpu().numpy(), ids, vocab)
        assert (np.abs(grad.double().cpu().numpy() - sums) <= (count[:, None] + 1) * U * size).all()
        want_v, want_x = sgd_f32.sgd_step(table.cpu().numpy(), grad.cpu().numpy(), v.cpu().numpy(), lr, mu)
        assert np.array_equal(v1.cpu().numpy(), want_v) and np.array_equal(x1.cpu().numpy(), want_x)
        table, v = x1, v1
