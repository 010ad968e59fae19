"""cn_embedding and cn_embedding_grad through the binding, against sums in 64 bits.

Tolerances.  Lookup: fp32 is one rounded product (2^-24 relative); 16-bit results are that product rounded once more
(2^-11 or 2^-8, and for fp16 half a step of 2^-24 below its normal range).  Gradient: a sum of n terms in fp32, in whatever
order, is off by at most (n - 1) roundings of partial sums no larger than the sum of magnitudes, the scaling and the addition
to what is there round once each, and a 16-bit result once more: (n + 2) 2^-24 (|scale| sum |dY| + |old|) + half a step."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HALF = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
SMALLEST = {"float32": 0.0, "float16": 2.0 ** -25, "bfloat16": 0.0}  # half a step below the normal range


@pytest.fixture(scope="module")
def torch():
    import torch
    import clusternet_amd as cn
    cn.init(0)
    return torch


def _tokens(torch, rng, rows, count, dtype, skew=True):
    """Frequent words first, some positions padded with numbers that name no row."""
    t = np.floor(np.exp(rng.uniform(0, np.log(rows + 1), count))).astype(np.int64) - 1 if skew else rng.integers(0, rows, count)
    t = np.clip(t, 0, rows - 1)
    if count > 4:
        t[rng.integers(0, count, max(1, count // 20))] = -1
        t[rng.integers(0, count, max(1, count // 50))] = rows
    return torch.from_numpy(t).to(getattr(torch, dtype)).cuda()


def _check_lookup(torch, table, tokens, scale, out):
    name = str(table.dtype).split(".")[1]
    t = tokens.long().cpu().flatten()
    named = (t >= 0) & (t < table.shape[0])
    want = torch.zeros(t.numel(), table.shape[1], dtype=torch.float64)
    s = float(np.float32(scale))
    want[named] = table.cpu().double()[t[named]] * s
    got = out.reshape(t.numel(), -1).cpu().double()
    assert out.dtype == table.dtype
    bound = want.abs() * (HALF[name] + 2.0 ** -24 * (1 + HALF[name])) + SMALLEST[name]
    assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() - bound).max())
    assert not got[~named].any()


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows,cols,count,index", [(1, 1, 1, "int64"), (7, 5, 3, "int32"), (100002, 120, 1408, "int64"),
                                                   (513, 64, 1023, "int32"), (300, 1001, 700, "int32"), (50, 4100, 33, "int64"),
                                                   (1000, 2048, 5000, "int32")])
def test_lookup(torch, dtype, rows, cols, count, index):
    import clusternet_amd as cn
    rng = np.random.default_rng(rows + cols + count)
    table = torch.from_numpy(rng.normal(0, 1, (rows, cols)).astype(np.float32)).cuda().to(getattr(torch, dtype))
    tokens = _tokens(torch, rng, rows, count, index)
    for scale in (1.0, 0.3, float(cols) ** 0.5):
        _check_lookup(torch, table, tokens, scale, cn.embedding(table, tokens, scale=scale))


def test_lookup_into_strided_and_unaligned_places(torch):
    """A table and an output that are parts of wider matrices, starting at odd elements; what surrounds the output stays."""
    import clusternet_amd as cn
    rng = np.random.default_rng(5)
    for dtype in (torch.float32, torch.bfloat16):
        for off, cols in ((0, 64), (1, 64), (3, 61)):
            wide = torch.from_numpy(rng.normal(0, 1, (400, 80)).astype(np.float32)).cuda().to(dtype)
            table = wide[:, off:off + cols]
            tokens = _tokens(torch, rng, 400, 333, "int32")
            back = torch.full((335, 90), 7.0, device="cuda", dtype=dtype)
            out = back[1:334, off + 2:off + 2 + cols]
            cn.embedding(table, tokens, scale=2.0, out=out)
            _check_lookup(torch, table, tokens, 2.0, out)
            keep = torch.ones_like(back, dtype=torch.bool)
            keep[1:334, off + 2:off + 2 + cols] = False
            assert bool((back[keep] == 7.0).all())


def test_lookup_shapes_and_tokens_beyond_32_bits(torch):
    import clusternet_amd as cn
    table = torch.arange(12, dtype=torch.float32, device="cuda").reshape(4, 3)
    far = torch.tensor([[0, 2 ** 32 + 1, -2 ** 32], [3, 4, 2 ** 62]], device="cuda")
    out = cn.embedding(table, far)
    assert out.shape == (2, 3, 3)
    assert torch.equal(out[0, 0], table[0]) and torch.equal(out[1, 0], table[3])
    assert not out[0, 1:].any() and not out[1, 1:].any()
    assert cn.embedding(table, far[:0]).shape == (0, 3, 3)
    # a table with values that are not finite, and padding that must stay zero under a scale that is not finite either
    table[1] = float("nan")
    table[2, 0] = float("inf")
    out = cn.embedding(table, torch.tensor([1, 2, -1], device="cuda", dtype=torch.int32), scale=float("inf"))
    assert bool(out[0].isnan().all()) and float(out[1, 0]) == float("inf") and not out[2].any()


def test_lookup_far_into_a_long_table(torch):
    """A row whose offset passes 2^31 elements, and one that passes 2^32 bytes."""
    import clusternet_amd as cn
    cols = 4096
    rows = (2 ** 31 + 2 ** 20) // cols
    table = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    table[-1] = 3.0
    table[rows // 2 + 1] = 5.0
    out = cn.embedding(table, torch.tensor([rows - 1, rows // 2 + 1, 0], device="cuda"), scale=1.0)
    assert bool((out[0] == 3.0).all()) and bool((out[1] == 5.0).all()) and not out[2].any()


def _grad_reference(torch, dY, tokens, rows, scale, old=None):
    t = tokens.long().cpu().flatten()
    named = (t >= 0) & (t < rows)
    d = dY.reshape(t.numel(), -1).cpu().double()
    s = float(np.float32(scale))
    want = torch.zeros(rows, d.shape[1], dtype=torch.float64) if old is None else old.cpu().double()
    mag = want.abs()
    want.index_add_(0, t[named], d[named] * s)
    mag.index_add_(0, t[named], (d[named] * s).abs())
    n = torch.zeros(rows, dtype=torch.float64).index_add_(0, t[named], torch.ones(int(named.sum()), dtype=torch.float64))
    return want, mag, n


def _check_grad(torch, dY, tokens, rows, scale, got, old=None):
    want, mag, n = _grad_reference(torch, dY, tokens, rows, scale, old)
    name = str(got.dtype).split(".")[1]
    bound = (n[:, None] + 2) * 2.0 ** -24 * mag
    if name != "float32":
        bound = bound * (1 + HALF[name]) + HALF[name] * want.abs() + SMALLEST[name]
    off = (got.cpu().double() - want).abs()
    assert bool((off <= bound).all()), float((off - bound).max())
    untouched = n == 0
    if old is None:
        assert not got.cpu()[untouched].any()
    else:
        assert torch.equal(got.cpu()[untouched], old.cpu()[untouched])


SIZES = [(1, 1, 1), (1, 3, 100), (7, 5, 3), (2, 16, 5000), (100002, 120, 1408), (513, 64, 8192), (513, 64, 8193),
         (300, 1001, 700), (3000, 33, 20000), (70000, 48, 70001), (600000, 8, 30000), (50, 4100, 333), (1000, 2048, 3000),
         (511, 16, 9000), (512, 16, 9000), (4000, 4, 131072), (4000, 4, 131073), (2 ** 20, 2, 300001),
         (999, 64, 2047), (999, 256, 2048), (999, 260, 2048), (999, 256, 2049), (999, 64, 1025), (5000, 61, 2048), (40, 512, 2000), (300, 255, 1500)]


@pytest.mark.parametrize("rows,cols,count", SIZES)
@pytest.mark.parametrize("dtype,to,index", [("float32", "float32", "int64"), ("float16", "float32", "int32"),
                                            ("float16", "float16", "int64"), ("bfloat16", "float32", "int32"),
                                            ("bfloat16", "bfloat16", "int32")])
def test_gradient(torch, rows, cols, count, dtype, to, index):
    import clusternet_amd as cn
    rng = np.random.default_rng(rows + cols + count)
    dY = torch.from_numpy(rng.normal(0, 1, (count, cols)).astype(np.float32)).cuda().to(getattr(torch, dtype))
    tokens = _tokens(torch, rng, rows, count, index)
    got = cn.embedding_grad(dY, tokens, rows, scale=0.7, out_dtype=getattr(torch, to))
    _check_grad(torch, dY, tokens, rows, 0.7, got)
    again = cn.embedding_grad(dY, tokens, rows, scale=0.7, out_dtype=getattr(torch, to))
    assert torch.equal(got, again)
    old = torch.from_numpy(rng.normal(0, 1, (rows, cols)).astype(np.float32)).cuda().to(getattr(torch, to))
    into = old.clone()
    assert cn.embedding_grad(dY, tokens, rows, scale=-0.1, out=into, accumulate=True) is into
    _check_grad(torch, dY, tokens, rows, -0.1, into, old)


@pytest.mark.parametrize("count", [1, 7, 8, 9, 64, 65, 2048, 2049, 4097, 30001])
@pytest.mark.parametrize("which", ["one token", "two in turn", "all padded", "each its own", "descending"])
@pytest.mark.parametrize("cols", [24, 600])
def test_gradient_of_extreme_texts(torch, count, which, cols):
    """Runs that fill every chunk, none, or exactly one; small whole numbers, so the sums are exact whatever their order."""
    import clusternet_amd as cn
    rows = 40000
    i = torch.arange(count, device="cuda")
    tokens = {"one token": i * 0 + 12345, "two in turn": (i % 2) * 39999, "all padded": i * 0 - 1, "each its own": (i * 7) % rows,
              "descending": rows - 1 - i % rows}[which].to(torch.int32)
    rng = np.random.default_rng(count)
    dY = torch.from_numpy(rng.integers(-8, 9, (count, cols)).astype(np.float32)).cuda()
    want, _, _ = _grad_reference(torch, dY, tokens, rows, 1.0)
    assert torch.equal(cn.embedding_grad(dY, tokens, rows).cpu().double(), want)


def test_gradient_in_strided_places(torch):
    """dY and dE as parts of wider matrices, aligned and not; what surrounds dE stays."""
    import clusternet_amd as cn
    rng = np.random.default_rng(9)
    for dtype in (torch.float32, torch.bfloat16):
        for off, cols in ((0, 64), (1, 64), (5, 63)):
            dY = torch.from_numpy(rng.normal(0, 1, (900, 96)).astype(np.float32)).cuda().to(dtype)[:, off:off + cols]
            tokens = _tokens(torch, rng, 500, 900, "int32")
            back = torch.full((502, 88), 7.0, device="cuda")
            out = back[1:501, 8 + off:8 + off + cols]
            cn.embedding_grad(dY, tokens, 500, scale=1.5, out=out)
            _check_grad(torch, dY, tokens, 500, 1.5, out)
            keep = torch.ones_like(back, dtype=torch.bool)
            keep[1:501, 8 + off:8 + off + cols] = False
            assert bool((back[keep] == 7.0).all())


def test_gradient_of_nothing(torch):
    import clusternet_amd as cn
    none = torch.empty(0, 12, device="cuda")
    tokens = torch.empty(0, dtype=torch.int64, device="cuda")
    out = torch.full((77, 12), 3.0, device="cuda")
    cn.embedding_grad(none, tokens, 77, out=out, accumulate=True)
    assert bool((out == 3.0).all())
    cn.embedding_grad(none, tokens, 77, out=out)
    assert not out.any()
    assert cn.embedding_grad(torch.empty(5, 0, device="cuda"), torch.zeros(5, dtype=torch.int32, device="cuda"), 3).shape == (3, 0)
    assert cn.embedding_grad(torch.ones(5, 4, device="cuda"), torch.zeros(5, dtype=torch.int32, device="cuda"), 0).shape == (0, 4)
    windows = torch.zeros(5, 3, dtype=torch.int32, device="cuda")
    assert cn.embedding_grad(torch.empty(5, 3, 0, device="cuda"), windows, 7).shape == (7, 0)
    assert not cn.embedding_grad(torch.empty(0, 3, 4, device="cuda"), windows[:0], 7).any()
    assert torch.equal(cn.embedding_grad(torch.ones(4, device="cuda"), windows[0, 0], 2), torch.tensor([[1.0] * 4, [0.0] * 4], device="cuda"))
    with pytest.raises(ValueError):  # rows of a window lie apart in another way than windows do
        cn.embedding_grad(torch.ones(5, 4, 3, device="cuda")[:, :3], windows, 7)


def test_a_row_that_is_not_finite_stays_its_own(torch):
    """Inf and NaN in the errors of one word and of padded positions reach that word's row only."""
    import clusternet_amd as cn
    count, cols = 3000, 40
    tokens = torch.arange(count, device="cuda", dtype=torch.int32) % 97
    tokens[tokens == 5] = -1
    dY = torch.ones(count, cols, device="cuda")
    dY[tokens == -1] = float("nan")
    dY[tokens == 11] = float("inf")
    got = cn.embedding_grad(dY, tokens, 97)
    assert bool(torch.isinf(got[11]).all()) and not got[5].any()
    rest = [r for r in range(97) if r not in (5, 11)]
    assert torch.equal(got[rest], torch.bincount(tokens[tokens >= 0].long(), minlength=97).float()[rest][:, None].expand(-1, cols))


def test_gradient_against_differences(torch):
    """The lookup is linear in its table: <dE, D> = <dY, lookup(E + D) - lookup(E)> for whole-number E, D and a power of two
    as scale, where every step is exact."""
    import clusternet_amd as cn
    rng = np.random.default_rng(3)
    rows, cols, count = 900, 56, 4000
    E, D = (torch.from_numpy(rng.integers(-9, 10, (rows, cols)).astype(np.float32)).cuda() for _ in range(2))
    dY = torch.from_numpy(rng.integers(-9, 10, (count, cols)).astype(np.float32)).cuda()
    tokens = _tokens(torch, rng, rows, count, "int64")
    moved = cn.embedding(E + D, tokens, scale=0.5) - cn.embedding(E, tokens, scale=0.5)
    dE = cn.embedding_grad(dY, tokens, rows, scale=0.5)
    assert float((dE.double() * D.double()).sum()) == float((dY.double() * moved.double()).sum())


def test_in_graphs_and_on_other_streams(torch):
    """Two captured graphs with eager work between their replays, each with workspaces of its own, and a call on a side
    stream: the eager results bit for bit, for new tokens copied into the captured ones."""
    import clusternet_amd as cn
    rng = np.random.default_rng(11)
    rows, cols = 5000, 72
    sets = []
    for count in (2000, 12000):
        dY = torch.from_numpy(rng.normal(0, 1, (count, cols)).astype(np.float32)).cuda()
        tokens = _tokens(torch, rng, rows, count, "int32")
        cn.embedding_grad(dY, tokens, rows)  # first use outside the capture
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = cn.embedding_grad(dY, tokens, rows)
            looked = cn.embedding(got, tokens, scale=2.0)
        sets.append((dY, tokens, graph, got, looked))
    side = torch.cuda.Stream()
    for _ in range(4):
        for dY, tokens, graph, got, looked in sets:
            tokens.copy_(_tokens(torch, rng, rows, tokens.numel(), "int32"))
            dY.mul_(-1.25)
            want = cn.embedding_grad(dY, tokens, rows)
            with torch.cuda.stream(side):
                side.wait_stream(torch.cuda.default_stream())
                beside = cn.embedding_grad(dY, tokens, rows)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want) and torch.equal(beside, want)
            assert torch.equal(looked, cn.embedding(want, tokens, scale=2.0))
