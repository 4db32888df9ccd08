"""Token embedding and its gradient on the GPU, against their definitions.  The lookup is one fp32
product and one rounding, so it is compared bit for bit; a gradient is a sum of k fp32 terms, which
in any order is off by at most (k - 1) 2^-24 times the sum of the magnitudes, then a product, a sum
with the old value and one rounding of the output's type."""
import numpy as np
import pytest
import torch

from oracle import vocab_f64

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
I32, I64 = torch.int32, torch.int64
U = 2.0 ** -24
HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}  # finfo.eps / 2
TINY = {F32: 2.0 ** -149, F16: 2.0 ** -25, BF16: 2.0 ** -133}


def _randn(*shape, dtype=F32, seed=0, std=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=gen) * std).to(dtype)


def _ids(n, rows, kind, seed=0):
    rng = np.random.default_rng([seed, n, rows])
    if kind == "same":
        return torch.full((n,), rows // 2, dtype=I64)
    if kind == "zipf":
        return torch.from_numpy(np.minimum(np.exp(rng.uniform(0, np.log(rows + 1), n)).astype(np.int64) - 1, rows - 1))
    if kind == "outside":
        return torch.from_numpy(rng.integers(-rows, 2 * rows, n))
    return torch.from_numpy(rng.integers(0, rows, n))


@pytest.mark.parametrize("ids_dtype", [I32, I64])
@pytest.mark.parametrize("out", [F32, F16, BF16])
@pytest.mark.parametrize("table", [F32, F16, BF16])
def test_lookup_types(native_libs, table, out, ids_dtype):
    from raf_amd import op

    for rows, width, n, scale in ((50, 24, 33, 3.3), (7, 513, 5, 1.0), (300, 1, 700, 0.1), (3, 7, 1, -2.0)):
        x, ids = _randn(rows, width, dtype=table, seed=n), _ids(n, rows, "outside", seed=1).to(ids_dtype)
        got = op.embedding(x.to(DEV), ids.to(DEV), scale=scale, out_dtype=out)
        inside = ((ids >= 0) & (ids < rows))[:, None]
        want = torch.where(inside, x[ids.long().clamp(0, rows - 1)].float() * np.float32(scale), torch.zeros(())).to(out)
        assert got.dtype == out and torch.equal(got.cpu(), want), (rows, width, n)


@pytest.mark.parametrize("width", [1, 2, 7, 8, 9, 63, 64, 65, 512, 1024, 1027, 1600, 4096, 8200])
def test_lookup_widths_lengths_and_shards(native_libs, width):
    from raf_amd import op

    x = _randn(90, width, seed=width)
    xd = x.to(DEV)
    for shape in ((1,), (3,), (2, 5), (257,), (4, 600)):
        n = int(np.prod(shape))
        ids = _ids(n, 90, "zipf", seed=2).reshape(shape)
        assert torch.equal(op.embedding(xd, ids.to(DEV)).cpu(), x[ids])
        shard = op.embedding(xd[30:70].contiguous(), ids.to(DEV), first_row=30).cpu()
        want = torch.where(((ids >= 30) & (ids < 70))[..., None], x[ids], torch.zeros(()))
        assert torch.equal(shard, want)


def test_lookup_of_nothing_and_extreme_indices(native_libs):
    from raf_amd import op

    x = _randn(5, 12).to(DEV)
    assert op.embedding(x, torch.zeros(0, dtype=I64, device=DEV)).shape == (0, 12)
    assert op.embedding(x, torch.zeros(2, 0, 3, dtype=I32, device=DEV)).shape == (2, 0, 3, 12)
    assert op.embedding(x[:, :0].contiguous(), torch.zeros(4, dtype=I64, device=DEV)).shape == (4, 0)
    assert not op.embedding(x[:0].contiguous(), torch.zeros(4, dtype=I64, device=DEV)).any()
    assert op.embedding(x, torch.tensor(3, device=DEV)).shape == (12,)
    info = torch.iinfo(I64)
    far = torch.tensor([info.min, info.max, -1, 5, 2 ** 32, 2 ** 32 + 1, -2 ** 31, 4], device=DEV)
    for first in (0, 4, 2 ** 40):
        got = op.embedding(x, far, scale=float("inf"), first_row=first)  # zeros whatever the scale
        inside = (far >= first) & (far - first < 5) if first < 2 ** 40 else torch.zeros(8, dtype=torch.bool, device=DEV)
        assert torch.equal(got.ne(0).any(1), inside)
    assert torch.equal(op.embedding(x, torch.tensor([2 ** 40 + 2], device=DEV), first_row=2 ** 40)[0], x[2])


def test_lookup_special_values_and_odd_addresses(native_libs):
    from raf_amd import op

    x = torch.tensor([[float("inf"), -float("inf"), float("nan"), -0.0, 65504.0, 1e-8, 3.0, 1.0, 2.0]])
    got = op.embedding(x.to(DEV), torch.zeros(2, dtype=I64, device=DEV), scale=2.0, out_dtype=F16).cpu()
    want = (x * 2).to(F16).expand(2, 9)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[~want.isnan()], want[~want.isnan()])
    assert torch.equal(torch.signbit(got[:, 3]), torch.tensor([True, True]))
    for dtype in (F16, BF16, F32):
        for off in (1, 2, 3):  # a table that starts anywhere, rows that start anywhere
            base = _randn(off + 20 * 51, dtype=dtype, seed=off).to(DEV)
            t = base[off:].view(20, 51)
            ids = _ids(77, 20, "uniform").to(DEV)
            assert torch.equal(op.embedding(t, ids), t[ids])


def test_lookup_and_gradient_beyond_2_to_31_elements(native_libs):
    """Rows whose element offset passes 2^31 (and whose byte offset passes 2^32)."""
    from raf_amd import op

    rows, width = 1_100_000, 2048
    x = torch.zeros(rows, width, dtype=BF16, device=DEV)
    ids = torch.tensor([rows - 1, 0, 1_048_576, 1_048_575, rows - 1] * 60, device=DEV)
    x[ids[:4]] = _randn(4, width, dtype=BF16).to(DEV)
    got = op.embedding(x, ids)
    assert torch.equal(got, x[ids])
    del x
    dy = torch.ones(300, width, dtype=BF16, device=DEV)
    dx = op.embedding_dx(dy, ids, rows)
    touched = dx.ne(0).any(1).nonzero().flatten()
    assert touched.tolist() == [0, 1_048_575, 1_048_576, rows - 1]
    assert dx[rows - 1].eq(120).all() and dx[1_048_576].eq(60).all()


def test_lookup_of_more_tokens_than_a_launch_holds(native_libs):
    """Rows of 513 words are a workgroup each, and 2^24 workgroups one more than a launch may have: the last
    tokens are another launch's."""
    from raf_amd import op

    n, rows, width = (1 << 24) + 5, 3, 4104
    if torch.cuda.mem_get_info()[0] < 2.2 * n * width:
        pytest.skip("needs 138 GB of free memory")
    x = _randn(rows, width, dtype=BF16).to(DEV)
    ids = torch.arange(n, device=DEV, dtype=I32) % 4  # 3 is outside
    y = op.embedding(x, ids)
    zero = torch.cat([x, torch.zeros(1, width, dtype=BF16, device=DEV)])
    for at in (0, 4_000_000, (1 << 24) - 1028, n - 1024):
        assert torch.equal(y[at:at + 1024], zero[ids[at:at + 1024].long()])
    del y
    torch.cuda.empty_cache()


def _check_dx(got, dy, ids, rows, scale=1.0, padding=None, first=0, old=None):
    want, size, count = vocab_f64.embedding_dx(dy.float().numpy(), ids.numpy(), rows, np.float32(scale), padding, first)
    out = got.dtype
    before = np.zeros_like(want) if old is None else old.double().numpy()
    bound = 1.01 * U * np.maximum(count, 1)[:, None] * size + 1.01 * U * (np.abs(want) + np.abs(want + before))
    bound += 1.01 * HALF_STEP[out] * (np.abs(want + before) + bound) + TINY[out]
    off = np.abs(got.double().cpu().numpy() - (want + before))
    worst = np.max(off / bound, initial=0)
    assert worst <= 1, f"{worst:.3f} of the bound"
    still = torch.from_numpy(count == 0)
    if old is None:
        assert not got.cpu()[still].any()
    else:
        assert torch.equal(got.cpu()[still], old[still])


@pytest.mark.parametrize("ids_dtype", [I32, I64])
@pytest.mark.parametrize("out", [F32, F16, BF16])
@pytest.mark.parametrize("dy_dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n", [40, 700])
def test_gradient_types(native_libs, n, dy_dtype, out, ids_dtype):
    from raf_amd import op

    rows, width, scale = 60, 27, 1.7
    dy, ids = _randn(n, width, dtype=dy_dtype, seed=3), _ids(n, rows, "outside", seed=4).to(ids_dtype)
    old = _randn(rows, width, dtype=out, seed=5)
    got = op.embedding_dx(dy.to(DEV), ids.to(DEV), rows, scale=scale, out_dtype=out)
    assert got.dtype == out
    _check_dx(got, dy, ids, rows, scale)
    grad = old.to(DEV)
    assert op.embedding_dx(dy.to(DEV), ids.to(DEV), rows, scale=scale, padding_idx=3, grad=grad) is grad
    _check_dx(grad, dy, ids, rows, scale, padding=3, old=old)


@pytest.mark.parametrize("kind", ["uniform", "zipf", "same", "outside"])
@pytest.mark.parametrize("n,rows,width", [
    (1, 10, 8), (2, 1, 5), (33, 40, 64), (64, 7, 9), (65, 7, 512), (255, 1000, 1), (256, 9, 1030),  # one launch
    (257, 1000, 8), (300, 3, 521), (2047, 5000, 16), (2048, 11, 24), (2049, 50257, 4), (5000, 200, 100),
    (20_000, 30522, 12), (70_000, 600, 3), (131_072, 5000, 2), (140_000, 2000, 1)])
def test_gradient_sizes(native_libs, kind, n, rows, width):
    """Calls of one launch and of four, tables of one row, long rows of one chunk, of several and of
    thousands, tiles of 2048 tokens and more."""
    from raf_amd import op

    dy, ids = _randn(n, width, dtype=BF16, seed=n), _ids(n, rows, kind, seed=6)
    dyd, idd = dy.to(DEV), ids.to(DEV)
    got = op.embedding_dx(dyd, idd, rows, out_dtype=F32)
    _check_dx(got, dy, ids, rows)
    for _ in range(2):  # equal bits, whatever order the long rows were listed in
        assert torch.equal(op.embedding_dx(dyd, idd, rows, out_dtype=F32), got)
    old = _randn(rows, width, dtype=F32, seed=8)
    _check_dx(op.embedding_dx(dyd, idd, rows, scale=-0.5, padding_idx=int(ids[0]), grad=old.to(DEV)), dy, ids, rows, -0.5,
              padding=int(ids[0]), old=old)


def test_gradient_of_many_rows_takes_many_tiles(native_libs):
    """A vocabulary so long that its keys leave room for small tiles only: more than 64 of them."""
    from raf_amd import op

    rows, n, width = 1_200_000, 300_000, 3
    rng = np.random.default_rng(9)
    ids = np.where(rng.random(n) < 0.5, rng.integers(0, rows, n), rng.choice([5, 1_199_999, 70_000, 70_001], n))
    dy = _randn(n, width, seed=10)
    got = op.embedding_dx(dy.to(DEV), torch.from_numpy(ids).to(DEV), rows).cpu().double()
    k = np.bincount(ids, minlength=rows)
    want = torch.zeros(rows, width, dtype=torch.float64).index_add_(0, torch.from_numpy(ids), dy.double())
    size = torch.zeros(rows, width, dtype=torch.float64).index_add_(0, torch.from_numpy(ids), dy.double().abs())
    bound = 1.01 * U * torch.from_numpy(np.maximum(k, 1))[:, None] * size + 3 * U * want.abs()
    assert bool(((got - want).abs() <= bound).all())
    assert k.max() > 30_000


@pytest.mark.parametrize("n", [1 << 16, 1 << 20, 1 << 22, 8_388_608])
def test_gradient_of_a_token_that_occurs_millions_of_times(native_libs, n):
    """A token's sum is off by the 31 additions of a chunk and its last rounding, however often it occurs;
    8,388,608 tokens are the most that are taken."""
    from raf_amd import op

    rows, value = 1000, torch.tensor([0.3, 0.7, 0.11, 1.3, -0.9])
    dy = value.expand(n, 5).contiguous().to(DEV)
    ids = torch.full((n,), 500, dtype=I32, device=DEV)
    ids[5::1000] = 3
    ids[7::1000] = -1
    got = op.embedding_dx(dy, ids, rows).cpu().double()
    for row in (3, 500):
        want = value.double() * int((ids == row).sum())
        assert ((got[row] - want).abs() <= 33 * U * want.abs()).all(), row
    got[[3, 500]] = 0
    assert not got.any()


def test_gradient_of_the_largest_batch(native_libs):
    from raf_amd import op

    n, rows, width = 8_388_608, 262_143, 3
    gen = torch.Generator(device=DEV).manual_seed(11)
    ids = (torch.exp(torch.rand(n, device=DEV, generator=gen, dtype=torch.float64) * np.log(rows)).long() - 1) % rows
    ids[::7] = torch.randint(0, rows, (len(ids[::7]),), device=DEV, generator=gen)
    dy = (torch.randn(n, width, device=DEV, generator=gen) * 1024).round() / 1024
    got = op.embedding_dx(dy, ids, rows).double()
    in_order, order = torch.sort(ids)
    ends = torch.searchsorted(in_order, torch.arange(rows + 1, device=DEV))

    def by_rows(x):  # differences of running sums, which are exact: multiples of 2^-10 below 2^26
        running = torch.cat([torch.zeros(1, width, device=DEV, dtype=torch.float64), x[order].double().cumsum(0)])
        return running[ends[1:]] - running[ends[:-1]]

    assert ((got - by_rows(dy)).abs() <= 33 * U * by_rows(dy.abs())).all()


def test_the_widest_rows(native_libs):
    """2^24 - 1 columns, a row beyond the reach of 32-bit byte offsets behind a few others."""
    from raf_amd import op

    rows, width = 70, (1 << 24) - 1
    x = torch.zeros(rows, width, dtype=F16, device=DEV)
    x[:, ::1_000_003] = _randn(rows, 17, dtype=F16).to(DEV)
    x[:, -1] = torch.arange(rows, dtype=F16, device=DEV) + 1
    for n in (3, 300):
        ids = torch.arange(n, dtype=I32, device=DEV) * 23 % (rows + 1)  # the last is outside
        y = op.embedding(x, ids)
        inside = ids < rows
        for at in range(0, n, max(n // 7, 1)):
            assert torch.equal(y[at], x[ids[at]]) if inside[at] else not y[at].any()
        dx = op.embedding_dx(y, ids, rows)
        count = torch.bincount(ids.long(), minlength=rows)[:rows]
        for row in range(0, rows, 9):  # sums of equal halves, a few of them: exact in fp32
            assert torch.equal(dx[row], (x[row].float() * count[row]).to(F16)), row
        assert torch.equal(dx[:, -1], ((torch.arange(rows, device=DEV) + 1) * count).to(F16))
        del y, dx
    del x
    torch.cuda.empty_cache()


def test_gradient_leaves_out_what_takes_no_part(native_libs):
    """Tokens of padding and of other shards: their gradients may hold anything."""
    from raf_amd import op

    rows, width, first = 50, 40, 100
    for n in (200, 3000):
        ids = _ids(n, 200, "uniform", seed=n)
        dy = _randn(n, width, seed=n)
        dead = (ids < first) | (ids >= first + rows) | (ids == 120)
        dy[dead] = float("nan")
        got = op.embedding_dx(dy.to(DEV), ids.to(DEV), rows, padding_idx=120, first_row=first)
        _check_dx(got, torch.where(dead[:, None], torch.zeros(()), dy), ids, rows, padding=120, first=first)
        all_dead = torch.full((n,), 120, device=DEV)
        assert not op.embedding_dx(dy.to(DEV), all_dead, rows, padding_idx=120, first_row=first).any()
        old = _randn(rows, width).to(DEV)
        assert torch.equal(op.embedding_dx(dy.to(DEV), all_dead, rows, padding_idx=120, first_row=first, grad=old.clone()), old)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("width", [1, 2, 3, 7, 8, 13, 520])
def test_gradient_of_few_rows_of_many(native_libs, width, dtype):
    """The gradient is zeroed as a whole first: from any element on, to the last, and nothing beside it."""
    from raf_amd import kernels

    n, rows = 300, 2411
    ids = _ids(n, rows, "zipf")
    dy = _randn(n, width, dtype=dtype)
    want, size, count = vocab_f64.embedding_dx(dy.float().numpy(), ids.numpy(), rows)
    for shift in range(0, 9, 2 if width > 8 else 1):
        room = torch.full((rows * width + 16,), float("nan"), dtype=dtype, device=DEV)
        out = room[shift:shift + rows * width].view(rows, width)
        kernels.embedding_dx(dy.to(DEV), ids.to(DEV), out)
        got = out.double().cpu().numpy()
        bound = count[:, None] * U * size + 1.01 * HALF_STEP[dtype] * (np.abs(want) + count[:, None] * U * size) + TINY[dtype]
        assert (np.abs(got - want) <= bound).all() and not got[count == 0].any()
        assert room[:shift].isnan().all() and room[shift + rows * width:].isnan().all()


def test_gradient_of_nothing(native_libs):
    from raf_amd import op

    none = torch.zeros(0, dtype=I64, device=DEV)
    assert not op.embedding_dx(torch.zeros(0, 9, device=DEV), none, 6).any()
    grad = _randn(6, 9).to(DEV)
    assert torch.equal(op.embedding_dx(torch.zeros(0, 9, device=DEV), none, 6, grad=grad.clone()), grad)
    assert op.embedding_dx(torch.zeros(5, 0, device=DEV), torch.zeros(5, dtype=I64, device=DEV), 6).shape == (6, 0)
    assert op.embedding_dx(torch.zeros(5, 3, device=DEV), torch.zeros(5, dtype=I64, device=DEV), 0).shape == (0, 3)


def test_gradient_propagates_inf_and_nan(native_libs):
    from raf_amd import op

    dy = torch.ones(400, 10)
    dy[3, 2], dy[5, 4], dy[7, 4] = float("inf"), float("inf"), -float("inf")
    ids = torch.zeros(400, dtype=I64)
    got = op.embedding_dx(dy.to(DEV), ids.to(DEV), 2).cpu()
    assert got[0, 2] == float("inf") and got[0, 4].isnan() and got[0, 0] == 400 and not got[1].any()


def test_gradient_against_differences(native_libs):
    """sum(dy * embedding(x)) is linear in the table: its difference quotient is the gradient."""
    from raf_amd import op

    rows, width, n = 12, 6, 500
    x, dy, ids = _randn(rows, width, seed=1).double(), _randn(n, width, seed=2), _ids(n, rows, "zipf")
    dx = op.embedding_dx(dy.to(DEV), ids.to(DEV), rows, scale=2.0).cpu().double()
    value = lambda t: float((vocab_f64.embedding(t.numpy(), ids.numpy(), 2.0) * dy.double().numpy()).sum())
    for at in ((0, 0), (3, 5), (11, 2)):
        up = x.clone()
        up[at] += 1.0
        assert float(dx[at]) == pytest.approx(value(up) - value(x), abs=1e-4)


def test_streams_and_graphs(native_libs):
    """Calls on a side stream, and a captured lookup and gradient replayed with new contents."""
    from raf_amd import op

    rows, width, n = 3000, 72, 4100
    x, dy = _randn(rows, width).to(DEV), _randn(n, width, dtype=BF16).to(DEV)
    ids = _ids(n, rows, "zipf").to(DEV)
    want = op.embedding(x, ids, scale=3.0), op.embedding_dx(dy, ids, rows, out_dtype=F32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = op.embedding(x, ids, scale=3.0), op.embedding_dx(dy, ids, rows, out_dtype=F32)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):  # two graphs: neither disturbs the other's workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = op.embedding(x, ids, scale=3.0), op.embedding_dx(dy, ids, rows, out_dtype=F32)
        graphs.append((graph, out))
    for k in range(4):
        ids.copy_(_ids(n, rows, ("zipf", "same", "outside", "uniform")[k], seed=k).to(DEV))
        dy.copy_(_randn(n, width, dtype=BF16, seed=k + 20).to(DEV))
        want = op.embedding(x, ids, scale=3.0), op.embedding_dx(dy, ids, rows, out_dtype=F32)
        torch.cuda.synchronize()
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want)), k


def test_two_threads_share_an_operator(native_libs):
    import threading

    from raf_amd import op

    rows, width, n = 500, 33, 2500
    work = []
    for k in range(2):
        dy, ids = _randn(n, width, seed=k).to(DEV), _ids(n, rows, "zipf", seed=k).to(DEV)
        work.append((dy, ids, op.embedding_dx(dy, ids, rows)))
    torch.cuda.synchronize()
    bad = []

    def go(k):
        dy, ids, want = work[k]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                if not torch.equal(op.embedding_dx(dy, ids, rows), want):
                    bad.append(k)

    threads = [threading.Thread(target=go, args=(k,)) for k in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


def test_direct_handles_agree(native_libs):
    from raf_amd import kernels, op

    x, ids = _randn(40, 30).to(DEV), _ids(600, 60, "uniform").to(DEV)
    assert torch.equal(kernels.embedding(x, ids, 2.0, 5), op.embedding(x, ids, 2.0, 5))
    out = torch.empty(600, 30, dtype=BF16, device=DEV)
    assert torch.equal(kernels.embedding(x, ids, out=out), op.embedding(x, ids, out_dtype=BF16))
    dy = _randn(600, 30).to(DEV)
    dx = torch.full((40, 30), 7.0, device=DEV)
    kernels.embedding_dx(dy, ids, dx, scale=2.0, padding_idx=9, first_row=5)
    assert torch.equal(dx, op.embedding_dx(dy, ids, 40, scale=2.0, padding_idx=9, first_row=5))
    with pytest.raises(ValueError):
        kernels.embedding_dx(dy, ids, dx[:, :29].contiguous())
    with pytest.raises(ValueError):
        kernels.embedding(x, ids, out=out[:599])
    with pytest.raises(TypeError):
        kernels.embedding(x.double(), ids)


def test_refusals_on_the_device(native_libs):
    from raf_amd import _lib, op

    x, ids = _randn(4, 8).to(DEV), torch.zeros(3, dtype=I64, device=DEV)
    with pytest.raises(_lib.RafError, match="unsupported dtype of x"):
        op.embedding(x.double(), ids)
    with pytest.raises(_lib.RafError, match="unsupported dtype of the output"):
        op.embedding(x, ids, out_dtype=torch.float64)
    with pytest.raises(_lib.RafError, match="different devices"):
        op.embedding(x, ids.cpu())
    with pytest.raises(_lib.RafError, match="unsupported sizes"):
        op.embedding_dx(torch.zeros(3, 1, device=DEV), ids, 1 << 21)


def test_a_gradient_that_is_its_own_input_is_refused(native_libs):
    from raf_amd import _lib, kernels, op

    for n in (40, 3000):
        dy, ids = _randn(n, 16).to(DEV), _ids(n, n, "uniform").to(DEV)
        with pytest.raises(_lib.RafError, match="dx overlaps dy"):
            op.embedding_dx(dy, ids, n, grad=dy)
        room = torch.zeros(2 * n, 16, device=DEV)
        with pytest.raises(_lib.RafError, match="dx overlaps dy"):  # by one row
            op.embedding_dx(room[:n], ids, n, grad=room[n - 1:-1])
        _check_dx(op.embedding_dx(room[:n].copy_(dy), ids, n, grad=room[n:]), dy.cpu(), ids.cpu(), n,
                  old=torch.zeros(n, 16))  # side by side
        bits = torch.zeros(n, 16, dtype=I32, device=DEV)  # the gradient within the indices' memory
        with pytest.raises(_lib.RafError, match="dx overlaps indices"):
            op.embedding_dx(dy, bits.view(-1)[:n], n, grad=bits.view(F32))
        with pytest.raises(ValueError, match="overlaps"):
            kernels.embedding_dx(dy, ids, dy)


def test_direct_handles_refuse_integers_beyond_64_bits(native_libs):
    from raf_amd import kernels

    x, ids, dx = _randn(5, 8).to(DEV), torch.zeros(3, dtype=I64, device=DEV), torch.zeros(5, 8, device=DEV)
    for call in (lambda: kernels.embedding(x, ids, first_row=1 << 64),
                 lambda: kernels.embedding_dx(x[:3], ids, dx, first_row=1 << 64),
                 lambda: kernels.embedding_dx(x[:3], ids, dx, padding_idx=1 << 64)):
        with pytest.raises(ValueError, match="does not fit 64 bits"):
            call()
