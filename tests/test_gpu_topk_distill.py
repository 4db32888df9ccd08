"""Distillation against a teacher's top logits on the GPU, against its definition in float64.

Bounds.  With u = 2^-24, each exponential of an argument x (in powers of two) is off relatively by
the rounding of its argument, at most 4 u |x| with the constant's, and 2 u of its own; a sum of V of
them by the longest chain of additions a column passes through, at most 256 here (columns per
thread, wavefront, workgroup, parts), and the logarithm's rounding by u |log S| (and log2 V more in
the exponent of a softmax).  E = 300 + 8 (max |z - m| / T log2 e + log2 V) collects these, in units
of u, for every softmax value, probability of the teacher and log sum; a gradient is a sum of such
values and one rounding of its type, a loss a sum of such logarithms times its weights."""
import numpy as np
import pytest
import torch

from oracle import vocab_f64

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
I32, I64 = torch.int32, torch.int64
U = 2.0 ** -24
HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F32: 2.0 ** -126, F16: 2.0 ** -25, BF16: 2.0 ** -126}  # exp2 flushes what is below the normal range
INF = float("inf")


def _case(rows, vocab, k, dtype=F32, teacher=F32, ids=I64, seed=0, padded=0, absent=0.2, masked=0.2):
    rng = np.random.default_rng([seed, rows, vocab, k])
    z = torch.from_numpy(rng.normal(0, 2, (rows, vocab + padded)).astype(np.float32)).to(dtype)
    idx = rng.integers(0, max(vocab, 1), (rows, k))
    if k and vocab:
        z[torch.arange(rows)[:, None], torch.from_numpy(idx)] += 5
    t = torch.from_numpy(rng.normal(5, 2, (rows, k)).astype(np.float32)).to(teacher)
    idx[rng.random((rows, k)) < absent] = -1
    labels = rng.integers(0, max(vocab, 1), rows)
    off = rng.random(rows) < masked
    idx[off] = -1
    labels[off] = -100
    if k and not off.all():
        labels[~off] = np.where(rng.random((~off).sum()) < 0.5, idx[~off, 0], labels[~off])
    dloss = torch.from_numpy(rng.uniform(0.2, 1.5, rows).astype(np.float32))
    return z, torch.from_numpy(idx).to(ids), t, torch.from_numpy(labels).to(ids), dloss


def _want(z, idx, t, dloss, vocab, temperature, soft, labels, hard):
    with np.errstate(all="ignore"):
        zz = z[:, :vocab].double().numpy()
        r = vocab_f64.topk_distill(zz, idx.numpy(), t.double().numpy(), np.float32(temperature), np.float32(soft),
                                   None if labels is None else labels.numpy(), np.float32(hard), dloss.double().numpy())
        finite = np.where(np.isfinite(zz), zz, np.nan)
        spread = (np.nanmax(finite, 1, initial=-1e30) - np.nanmin(finite, 1, initial=1e30)) * max(1.0, 1.0 / temperature) * 1.4427
        spread = np.clip(spread, 0, 160)  # what lies further down is below the smallest number
    # An exponential below 2^-126 becomes 0 before its factor dloss soft T / S_T (or dloss hard / S_1; S >= 1)
    # enters: its element of the gradient is off by 2^-126 times that factor, not by 2^-126.
    r["factor"] = np.maximum(1.0, np.abs(dloss.double().numpy()) * (abs(soft) * temperature + abs(hard)))[:, None]
    r["E"] = 300 + 8 * (spread + np.log2(max(vocab, 2)))
    return r


def _check_loss(loss, r, temperature, soft, hard):
    got, want = loss.double().cpu().numpy().ravel(), r["loss"]
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isinf(got), np.isinf(want))
    with np.errstate(all="ignore"):
        bound = U * r["E"] * (abs(soft) * temperature ** 2 * (2 + 2 * r["cross"]) + 2 * abs(hard)) + 1.01 * U * np.abs(want)
        worst = np.max(np.nan_to_num(np.abs(got - want) / bound, nan=0, posinf=0), initial=0)
    assert worst <= 1, f"loss: {worst:.3f} of the bound"


def _check_stats(stats, r):
    got, want = stats.double().cpu().numpy().reshape(-1, 3), r["stats"]
    assert np.array_equal(got[:, 0], want[:, 0], equal_nan=True)  # the largest logit is one of them
    with np.errstate(all="ignore"):
        off = np.abs(got[:, 1:] - want[:, 1:])
    ok = (off <= U * r["E"][:, None] + 1.01 * U * np.abs(want[:, 1:])) | (np.isnan(got[:, 1:]) & np.isnan(want[:, 1:]))
    assert ok.all()


def _check_grad(grad, r, vocab):
    got = grad.cpu().reshape(-1, grad.shape[-1])
    assert not got[:, vocab:].any()  # padding columns
    got, want, out = got[:, :vocab].double().numpy(), r["dlogits"], grad.dtype
    assert np.array_equal(np.isnan(got), np.isnan(want))
    with np.errstate(all="ignore"):
        bound = U * r["E"][:, None] * (r["soft"] + r["p"] + r["hard"])
        bound += 1.01 * HALF_STEP[out] * (np.abs(want) + bound) + TINY[out] + 2.0 ** -126 * r["factor"]
        worst = np.max(np.nan_to_num(np.abs(got - want) / bound, nan=0), initial=0)
    assert worst <= 1, f"gradient: {worst:.3f} of the bound"


def _all(z, idx, t, labels, dloss, vocab=None, temperature=1.0, soft=1.0, hard=0.0):
    """The three operators on one case, each against the definition."""
    from raf_amd import op

    vocab = z.shape[1] if vocab is None else vocab
    r = _want(z, idx, t, dloss, vocab, temperature, soft, labels, hard)
    zd, idxd, td, dl = z.to(DEV), idx.to(DEV), t.to(DEV), dloss.to(DEV)
    ld = labels.to(DEV) if labels is not None else None
    more = dict(temperature=temperature, soft_weight=soft, labels=ld, hard_weight=hard, vocab_size=vocab)
    loss, stats = op.topk_distill(zd, idxd, td, **more)
    _check_loss(loss, r, temperature, soft, hard)
    _check_stats(stats, r)
    grad = op.topk_distill_dx(dl, zd, idxd, td, stats, **more)
    assert grad.dtype == z.dtype and grad.shape == z.shape
    _check_grad(grad, r, vocab)
    loss2, grad2 = op.topk_distill_step(zd, idxd, td, dl, **more)
    _check_loss(loss2, r, temperature, soft, hard)
    _check_grad(grad2, r, vocab)
    for again, first in zip(op.topk_distill_step(zd, idxd, td, dl, **more), (loss2, grad2)):
        assert torch.equal(again.view(torch.uint8), first.view(torch.uint8))
    assert torch.equal(zd.cpu().view(torch.uint8), z.view(torch.uint8))  # the logits are only read
    return loss, stats, grad, loss2, grad2


@pytest.mark.parametrize("ids", [I32, I64])
@pytest.mark.parametrize("teacher", [F32, F16, BF16])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_types(native_libs, dtype, teacher, ids):
    z, idx, t, labels, dloss = _case(37, 1003, 9, dtype, teacher, ids, padded=21)
    _all(z, idx, t, labels, dloss, vocab=1003, temperature=2.0, soft=0.8, hard=0.3)


@pytest.mark.parametrize("temperature,soft,hard,labelled", [
    (1.0, 1.0, 0.0, False), (1.0, 1.0, 0.0, True), (3.0, 1.0, 0.0, True), (1.0, 0.5, 0.5, True), (0.25, 1.0, 1.5, True),
    (5.0, 0.0, 1.0, True), (2.0, 0.0, 0.0, True), (2.0, -1.0, 0.5, True), (2.0, 1.0, 0.5, False)])
def test_weights_and_temperatures(native_libs, temperature, soft, hard, labelled):
    z, idx, t, labels, dloss = _case(19, 700, 5, BF16)
    _all(z, idx, t, labels if labelled else None, dloss, temperature=temperature, soft=soft, hard=hard)


@pytest.mark.parametrize("rows, vocab", [(21, 900), (600, 300), (3, 40_000), (70, 30_000)])
@pytest.mark.parametrize("temperature", [2.0, 4.0, 2.5])
def test_both_terms(native_libs, temperature, rows, vocab):
    """Two sums of one pass; at 2 and 4 the second is a power of the first.  The rows' ranges differ widely."""
    z, idx, t, labels, dloss = _case(rows, vocab, 5, F32)
    z *= torch.logspace(-3, 2, rows)[:, None]
    _all(z, idx, t, labels, dloss, temperature=temperature, hard=0.75)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab", [
    (5, 1), (5, 2), (3, 7), (3, 8), (4, 9), (9, 63), (600, 65), (7, 4096), (7, 4097), (1, 8191), (2, 8193), (1, 50257),
    (3, 50257), (515, 4999), (513, 16385), (2, 65537), (2, 131_073), (1, 200_003)])
def test_sizes(native_libs, rows, vocab, dtype):
    """One workgroup a row and several, rows in one to sixteen words a thread and rows too long for that."""
    z, idx, t, labels, dloss = _case(rows, vocab, 6, dtype, masked=0.1)
    _all(z, idx, t, labels, dloss, temperature=2.0, hard=0.25)


@pytest.mark.parametrize("rows", [515, 3])
@pytest.mark.parametrize("k", [0, 1, 2, 63, 64, 65, 300, 1024])
def test_teacher_lengths(native_libs, k, rows):
    z, idx, t, labels, dloss = _case(rows, 1500 if rows > 3 else 9000, k, F16)
    _all(z, idx, t, labels, dloss, temperature=1.5, hard=0.5)


@pytest.mark.parametrize("rows, vocab, dtype", [(520, 100_000, F32), (520, 90_001, F32), (100, 90_001, F32),
                                                (520, 204_808, BF16), (520, 204_807, F16), (520, 102_407, BF16), (65, 205_001, F16),
                                                (64, 70_001, F32), (64, 25_000, BF16), (64, 24_576, F16)])
def test_long_rows(native_libs, rows, vocab, dtype):
    """Rows that 256, 512 and 1024 threads hold in registers, the longest of each, and ones that none hold."""
    z, idx, t, labels, dloss = _case(rows, vocab, 4, dtype, masked=0.3)
    _all(z, idx, t, labels, dloss, temperature=2.0, hard=0.5)


def test_a_row_too_long_for_registers_among_many(native_libs):
    z, idx, t, labels, dloss = _case(520, 66_000, 4, F32, masked=0.3)
    _all(z, idx, t, labels, dloss, temperature=2.0)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows, temperature", [(65, 2.0), (65, 1.5), (65, 1.0), (520, 2.0), (3, 2.0)])
def test_sums_over_very_many_columns(native_libs, rows, temperature, dtype):
    """Rows of millions of equal columns behind larger ones (which every thread meets first, so that the others
    count less than one each): no thread's chain of additions grows with the row beyond what the bound
    above counts."""
    from raf_amd import op

    vocab, first = 1 << (24 if rows < 100 else 21), 1 << 15
    low = torch.tensor(-1.2).to(dtype)
    z = torch.full((rows, vocab), float(low), dtype=dtype, device=DEV)
    z[:, :first] = 0.0
    at = torch.arange(rows, device=DEV)
    more = dict(temperature=temperature, labels=at, hard_weight=1.0)
    loss, stats = op.topk_distill(z, at[:, None], torch.zeros(rows, 1, device=DEV), **more)
    want = [np.log(first + (vocab - first) * np.exp(float(low.double()) / t)) for t in (temperature, 1.0)]
    bound = U * (300 + 8 * (1.21 * 1.4427 + np.log2(vocab)))
    assert not stats[:, 0].any()
    for k in range(2):
        assert ((stats[:, k + 1].double() - want[k]).abs() <= bound + 1.01 * U * want[k]).all()
    total = temperature ** 2 * want[0] + want[1]
    assert ((loss.double() - total).abs() <= bound * (temperature ** 2 + 1) + 1.01 * U * total).all()


def test_more_rows_than_a_grid_dimension_holds(native_libs):
    z, idx, t, labels, dloss = _case(66_000, 3, 2, F32)
    _all(z, idx, t, labels, dloss, temperature=2.0, hard=1.0)


@pytest.mark.parametrize("rows", [1, 65])
def test_the_longest_rows(native_libs, rows):
    """2^28 - 1 columns, read in parts and whole: a uniform student, a teacher with the last column."""
    from raf_amd import op

    vocab = (1 << 28) - 1
    if torch.cuda.mem_get_info()[0] < 5 * rows * vocab:
        pytest.skip("needs 87 GB of free memory")
    z = torch.zeros(rows, vocab, dtype=BF16, device=DEV)
    idx = torch.tensor([[vocab - 1, 0, vocab]], dtype=I32, device=DEV).repeat(rows, 1)  # the third is outside
    t = torch.tensor([[2.0, 0.0, 9.0]], device=DEV).repeat(rows, 1)
    labels = torch.full((rows,), vocab - 2, dtype=I32, device=DEV)
    p = torch.softmax(t[0, :2].double() / 2, 0).cpu()
    more = dict(temperature=2.0, labels=labels, hard_weight=0.5)
    bound = U * (300 + 8 * 28)
    want = 4 * (float((p * p.log()).sum()) + np.log(vocab)) + 0.5 * np.log(vocab)
    loss, stats = op.topk_distill(z, idx, t, **more)
    assert ((loss.double() - want).abs() <= bound * 5 + 2 * U * want).all()
    assert ((stats[:, 1:].double() - np.log(vocab)).abs() <= bound + U * 20).all() and not stats[:, 0].any()
    one = torch.ones(1, device=DEV)

    def check(grad):
        for at, value in ((vocab - 1, -2 * p[0]), (0, -2 * p[1]), (vocab - 2, -0.5), (vocab // 2, 2.5 / vocab), (1, 2.5 / vocab)):
            near = 1.01 * HALF_STEP[BF16] * abs(float(value)) + 3 / vocab  # the two softmaxes where a target is
            assert ((grad[:, at].double() - float(value)).abs() <= near).all(), at
        assert (grad[:, 1:vocab - 2] == grad[0, 1]).all() and grad[0, 1] > 0

    check(op.topk_distill_dx(one, z, idx, t, stats, **more))
    loss2, grad = op.topk_distill_step(z, idx, t, one, **more)
    assert ((loss2.double() - want).abs() <= bound * 5 + 2 * U * want).all()
    check(grad)
    del z, grad
    torch.cuda.empty_cache()


def test_more_rows_than_a_launch_holds(native_libs):
    """2^24 workgroups of 256 threads are one more than a launch may have: the loss and the combined call go on
    in another.  Two columns, so that the definition is a formula; each rounding is at most 2^-24 of
    values below 16, and there are fewer than 64 of them."""
    from raf_amd import op

    rows = (1 << 24) + 77
    gen = torch.Generator(device=DEV).manual_seed(5)
    z = torch.randn(rows, 2, device=DEV, generator=gen)
    idx = torch.randint(-1, 2, (rows, 1), device=DEV, generator=gen, dtype=I32)
    idx[-77:] = torch.arange(77, device=DEV, dtype=I32)[:, None] % 2
    t = torch.randn(rows, 1, device=DEV, generator=gen)
    dloss = torch.rand(rows, device=DEV, generator=gen) + 0.5
    live = (idx >= 0).flatten()
    z64 = z.double()
    logq = torch.log_softmax(z64, 1)
    hot = torch.nn.functional.one_hot(idx.flatten().clamp(min=0).long(), 2)
    want = -(logq * hot).sum(1) * live
    grad = ((logq.exp() - hot) * dloss.double()[:, None]) * live[:, None]
    loss, stats = op.topk_distill(z, idx, t)
    assert ((loss - want).abs() <= 64 * U * 16).all() and not loss[~live].any()
    assert torch.equal(stats[:, 0], z.max(1).values * live)
    loss2, got = op.topk_distill_step(z, idx, t, dloss)
    assert ((loss2 - want).abs() <= 64 * U * 16).all() and ((got - grad).abs() <= 64 * U * 16).all()
    got = op.topk_distill_dx(dloss, z, idx, t, stats)
    assert ((got - grad).abs() <= 64 * U * 16).all()


def test_the_same_index_twice(native_libs):
    for rows, vocab in ((40, 300), (2, 20_000)):
        for k in (2, 50, 700):
            z, idx, t, labels, dloss = _case(rows, vocab, k, F32, absent=0.1, masked=0.0)
            idx = idx % 5  # -1 becomes 4
            labels = labels % 5
            _all(z, idx, t, labels, dloss, temperature=2.0, hard=0.7)


def test_rows_without_targets_are_not_looked_at(native_libs):
    for rows, vocab in ((600, 130), (4, 9001)):
        z, idx, t, labels, dloss = _case(rows, vocab, 4, F32, masked=0.0)
        dead = torch.arange(rows) % 2 == 1
        z[dead] = float("nan")
        idx[dead] = -1
        t[dead] = float("nan")
        labels[dead] = vocab  # outside, too
        loss, stats, grad, loss2, grad2 = _all(z, idx, t, labels, dloss, temperature=2.0, hard=0.5)
        for x in (loss, stats, grad, loss2, grad2):
            assert not x.cpu()[dead].any()


def test_infinities_and_lowest_values(native_libs):
    low = {F32: torch.finfo(F32).min, F16: torch.finfo(F16).min, BF16: torch.finfo(BF16).min}
    for dtype in (F32, F16, BF16):
        for vocab in (40, 9001):
            z, idx, t, labels, dloss = _case(7, vocab, 5, dtype, absent=0.0, masked=0.0)
            z[0, 10:] = -INF  # a masked vocabulary: the targets stay inside
            idx[0] = torch.arange(5)
            labels[0] = 9
            z[1, 10:] = low[dtype]
            idx[1] = torch.arange(5)
            labels[1] = 0
            z[2] = low[dtype]  # nothing stands out: uniform
            z[3, 3] = -INF  # a target that the student cannot give
            idx[3, 0] = 3
            z[4] = -INF  # nothing is left
            z[5, 2] = INF
            t[6, 1:4] = -INF  # entries that the teacher rules out
            t[6, 0] = low[F32]
            for temperature in (1.0, 2.0):
                loss, stats, grad, loss2, grad2 = _all(z, idx, t, labels, dloss, temperature=temperature, hard=0.5)
                assert loss[3].item() == INF and loss[4].isnan() and loss[5].isnan()
                assert torch.isfinite(grad[:3].float()).all()
    # a teacher that rules everything out is no teacher
    z, idx, t, labels, dloss = _case(3, 50, 4, F32, absent=0, masked=0)
    t[1] = -INF
    loss = _all(z, idx, t, None, dloss)[0]
    assert loss[1] == 0


def test_nan_in_a_live_row_stays_in_it(native_libs):
    z, idx, t, labels, dloss = _case(6, 5000, 4, BF16, absent=0, masked=0)
    z[2, 4321] = float("nan")
    t[4, 1] = float("nan")
    loss, stats, grad, loss2, grad2 = _all(z, idx, t, labels, dloss, hard=0.5)
    assert loss.isnan().tolist() == [False, False, True, False, True, False]


def test_large_logits_keep_their_softmax(native_libs):
    """The maximum and the log sum are kept apart: a common offset changes nothing."""
    from raf_amd import op

    z, idx, t, labels, dloss = _case(50, 3000, 8, F32, masked=0)
    z = (z * 64).round() / 64  # so that adding 2^17 is exact
    far = z + 2.0 ** 17
    a, b = (_all(x, idx, t, labels, dloss, temperature=2.0, hard=0.3) for x in (z, far))
    assert torch.equal(a[2], b[2]) and torch.equal(a[4], b[4])


def test_upstream_gradient_of_one_element_and_of_zero(native_libs):
    from raf_amd import op

    z, idx, t, labels, _ = _case(30, 800, 6, F32)
    one = torch.tensor([0.37])
    _all_one = _want(z, idx, t, one.expand(30), 800, 2.0, 1.0, None, 0.0)
    zd, idxd, td = z.to(DEV), idx.to(DEV), t.to(DEV)
    loss, stats = op.topk_distill(zd, idxd, td, temperature=2.0)
    for dl in (one, one.reshape(()), one.reshape(1, 1)):
        _check_grad(op.topk_distill_dx(dl.to(DEV), zd, idxd, td, stats, temperature=2.0), _all_one, 800)
        _check_grad(op.topk_distill_step(zd, idxd, td, dl.to(DEV), temperature=2.0)[1], _all_one, 800)
    zero = torch.zeros(30, device=DEV)
    assert not op.topk_distill_dx(zero, zd, idxd, td, stats, temperature=2.0).any()
    assert not op.topk_distill_step(zd, idxd, td, zero, temperature=2.0)[1].any()


@pytest.mark.parametrize("rows, vocab", [(37, 3000), (600, 3000), (5, 30_000)])
@pytest.mark.parametrize("temperature", [1.0, 1.5, 2.0, 4.0])
def test_upstream_gradient_of_any_magnitude(native_libs, temperature, rows, vocab):
    """A power of two in dloss changes nothing but the exponents, as long as the gradient is within fp32's range."""
    from raf_amd import op

    z, idx, t, labels, dloss = (x.to(DEV) for x in _case(rows, vocab, 6, F32))
    more = dict(temperature=temperature, labels=labels, hard_weight=0.5)
    loss, stats = op.topk_distill(z, idx, t, **more)
    for grad in (lambda dl: op.topk_distill_dx(dl, z, idx, t, stats, **more), lambda dl: op.topk_distill_step(z, idx, t, dl, **more)[1]):
        want = grad(dloss)
        for scale in (2.0 ** 118, 2.0 ** -40):
            got = grad(dloss * scale)
            assert torch.isfinite(got).all() and torch.equal(got / scale, want)


def test_gradient_against_differences(native_libs):
    """The row losses of the kernel itself, moved by a step in single logits."""
    from raf_amd import op

    z, idx, t, labels, dloss = _case(4, 40, 3, F32, masked=0)
    more = dict(temperature=2.0, labels=labels.to(DEV), hard_weight=0.5)
    value = lambda zz: (op.topk_distill(zz.to(DEV), idx.to(DEV), t.to(DEV), **more)[0].cpu().double() * dloss.double()).sum()
    grad = op.topk_distill_step(z.to(DEV), idx.to(DEV), t.to(DEV), dloss.to(DEV), **more)[1].cpu()
    h = 2.0 ** -5
    for at in [(0, int(idx[0].max())), (1, 7), (2, int(labels[2])), (3, 39)]:
        up, down = z.clone(), z.clone()
        up[at] += h
        down[at] -= h
        # the quotient's own error: h^2 / 6 times a third derivative below 8, and the losses' rounding over h
        assert float((value(up) - value(down)) / (2 * h)) == pytest.approx(float(grad[at]), abs=h * h * 8 / 6 + 1e-4)


def test_leading_dimensions_and_empty_shapes(native_libs):
    from raf_amd import op

    z, idx, t, labels, dloss = (x.to(DEV) for x in _case(24, 90, 4, F16))
    flat = op.topk_distill_step(z, idx, t, dloss, labels=labels, hard_weight=0.5)
    shaped = op.topk_distill_step(z.view(2, 3, 4, 90), idx.view(2, 3, 4, 4), t.view(2, 3, 4, 4), dloss.view(2, 3, 4),
                                  labels=labels.view(2, 3, 4), hard_weight=0.5)
    assert shaped[0].shape == (2, 3, 4) and torch.equal(shaped[0].flatten(), flat[0])
    assert shaped[1].shape == (2, 3, 4, 90) and torch.equal(shaped[1].view(24, 90), flat[1])
    one = op.topk_distill(z[0], idx[0], t[0])
    assert one[0].shape == () and one[1].shape == (3,)
    none = op.topk_distill_step(z[:0], idx[:0], t[:0], dloss[:0])
    assert none[0].shape == (0,) and none[1].shape == (0, 90)
    wide = op.topk_distill_step(z[:, :0].contiguous(), idx, t, dloss)
    assert not wide[0].any() and wide[1].shape == (24, 0)
    padded = op.topk_distill_step(z, idx, t, dloss, vocab_size=0)  # every column is padding
    assert not padded[0].any() and not padded[1].any()


def test_a_vocabulary_without_columns(native_libs):
    """Every column is padding: no loss, and a gradient of zeros as wide as it is asked for."""
    from raf_amd import kernels, op

    for rows in (24, 600):
        z, idx, t, labels, dloss = (x.to(DEV) for x in _case(rows, 90, 4, F16))
        more = dict(labels=labels, hard_weight=0.5, vocab_size=0)
        loss, stats = op.topk_distill(z, idx, t, **more)
        assert not loss.any() and not stats.any()
        assert not op.topk_distill_dx(dloss, z, idx, t, stats, **more).any()
        loss, grad = op.topk_distill_step(z, idx, t, dloss, **more)
        assert not loss.any() and not grad.any()
        h = kernels.TopkDistill(z[:, :0], idx, t, 2.0, 1.0, labels, 0.5)
        loss, stats = h.loss()
        assert not loss.any() and not stats.any()
        for width in (0, 1, 9, 515):
            wide = torch.full((rows, width), 9.0, dtype=F16, device=DEV)
            assert not h.dx(dloss, stats, out=wide).any()
            loss, grad = h.step(dloss, out=wide.fill_(9.0))
            assert not loss.any() and not grad.any()


def test_rows_of_a_wider_matrix(native_libs):
    """The direct handle takes rows that lie apart, and an output of another width than the input."""
    from raf_amd import kernels

    for dtype in (F16, F32):
        for stride, off in ((1010, 0), (1003, 3), (1001, 1)):
            for rows in (520, 5):
                z, idx, t, labels, dloss = _case(rows, 1000, 5, dtype)
                r = _want(z, idx, t, dloss, 1000, 2.0, 1.0, labels, 0.5)
                buf = torch.full((rows * stride + off,), float("nan"), dtype=dtype, device=DEV)
                view = buf[off:].view(rows, stride)[:, :1000]
                view.copy_(z)
                h = kernels.TopkDistill(view, idx.to(DEV), t.to(DEV), 2.0, 1.0, labels.to(DEV), 0.5)
                loss, stats = h.loss()
                _check_loss(loss, r, 2.0, 1.0, 0.5)
                out = torch.full((rows, 1007), 9.0, dtype=dtype, device=DEV)
                _check_grad(h.dx(dloss.to(DEV), stats, out=out), r, 1000)
                _check_grad(h.step(dloss.to(DEV), out=out.fill_(9.0))[1], r, 1000)
                assert bool(buf.isnan().sum() == buf.numel() - rows * 1000)


def test_rows_beyond_2_to_31_elements(native_libs):
    from raf_amd import op

    rows, vocab = 17_000, 130_000
    z = torch.zeros(rows, vocab, dtype=F16, device=DEV)
    idx = torch.full((rows, 2), -1, device=DEV)
    idx[[0, 16_600, rows - 1]] = torch.tensor([5, vocab - 1], device=DEV)
    t = torch.zeros(rows, 2, device=DEV)
    for loss, grad in (op.topk_distill_step(z, idx, t, torch.ones(1, device=DEV)),):
        assert loss.nonzero().flatten().tolist() == [0, 16_600, rows - 1]
        assert loss[rows - 1].item() == pytest.approx(np.log(vocab / 2), rel=1e-6)
        # minus a half, and the softmax's 1 / vocab, which is below the first's half step
        assert grad[[0, 16_600, rows - 1]][:, [5, vocab - 1]].eq(-0.5).all()
        assert grad[rows - 1, 6].item() == pytest.approx(1 / vocab, abs=2.0 ** -25) and not grad[1].any()
    loss2, stats = op.topk_distill(z, idx, t)
    assert torch.equal(loss2, loss)
    assert torch.equal(op.topk_distill_dx(torch.ones(1, device=DEV), z, idx, t, stats), grad)


def test_streams_and_graphs(native_libs):
    from raf_amd import op

    for rows, vocab in ((600, 2000), (3, 30_000)):
        z, idx, t, labels, dloss = (x.to(DEV) for x in _case(rows, vocab, 7, BF16))

        def calls():
            more = dict(temperature=2.0, labels=labels, hard_weight=0.5)
            loss, stats = op.topk_distill(z, idx, t, **more)
            return (loss, stats, op.topk_distill_dx(dloss, z, idx, t, stats, **more), *op.topk_distill_step(z, idx, t, dloss, **more))

        want = calls()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = calls()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = calls()
            graphs.append((graph, out))
        for k in range(3):
            for x, new in zip((z, idx, t, labels, dloss), _case(rows, vocab, 7, BF16, seed=k + 1)):
                x.copy_(new.to(DEV))
            want = calls()
            torch.cuda.synchronize()
            for graph, _ in graphs:
                graph.replay()
            torch.cuda.synchronize()
            for _, out in graphs:
                assert all(torch.equal(a, b) for a, b in zip(out, want)), k


def test_refusals_on_the_device(native_libs):
    from raf_amd import _lib, kernels, op

    z, idx, t, labels, dloss = (x.to(DEV) for x in _case(4, 50, 3))
    with pytest.raises(_lib.RafError, match="unsupported dtype of logits"):
        op.topk_distill(z.double(), idx, t)
    with pytest.raises(_lib.RafError, match="unsupported dtype of topk_logits"):
        op.topk_distill(z, idx, t.double())
    with pytest.raises(_lib.RafError, match="more than 1024"):
        op.topk_distill(z, torch.zeros(4, 1025, dtype=I64, device=DEV), torch.zeros(4, 1025, device=DEV))
    for temperature in (0.0, -2.0, float("nan"), INF):
        for call in (lambda: op.topk_distill(z, idx, t, temperature), lambda: op.topk_distill_step(z, idx, t, dloss, temperature),
                     lambda: op.topk_distill_dx(dloss, z, idx, t, torch.zeros(4, 3, device=DEV), temperature)):
            with pytest.raises(_lib.RafError, match="temperature"):
                call()
    with pytest.raises(_lib.RafError, match="different devices"):
        op.topk_distill(z, idx.cpu(), t)
    with pytest.raises(ValueError, match="neighbours"):
        kernels.TopkDistill(z.repeat(1, 2)[:, ::2], idx, t)
    with pytest.raises(ValueError, match="labels"):
        kernels.TopkDistill(z, idx, t, labels=labels[:3])
    with pytest.raises(ValueError, match="dloss"):
        kernels.TopkDistill(z, idx, t).step(dloss[:3])
    room = torch.zeros(4, 128, device=DEV)
    for out in (room, room.view(-1)[40:440].view(4, 100)):  # the logits' own memory, and part of it
        with pytest.raises(ValueError, match="overlaps"):
            kernels.TopkDistill(room[:, 50:100], idx, t).step(dloss, out=out)


def test_gradient_buffers_that_hold_another_input_are_refused(native_libs):
    from raf_amd import kernels

    for rows, vocab in ((30, 300), (600, 50)):
        z, idx, t, labels, dloss = (x.to(DEV) for x in _case(rows, vocab, 3))
        h = kernels.TopkDistill(z, idx, t, 2.0, 1.0, labels, 0.5)
        loss, stats = h.loss()
        out = torch.zeros(rows, vocab, device=DEV)
        of_rows, of_stats = out.view(-1)[5:5 + rows].copy_(dloss), out.view(-1)[-3 * rows:].view(rows, 3)
        for call in (lambda: h.step(of_rows, out=out), lambda: h.dx(of_rows, stats, out=out), lambda: h.dx(dloss, of_stats, out=out)):
            with pytest.raises(ValueError, match="overlaps"):
                call()
