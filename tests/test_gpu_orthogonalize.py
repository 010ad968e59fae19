"""cn_orthogonalize and cn_muon_update through the binding, against the same steps in 64 bits.

Tolerance.  A step maps singular values by p(s) = a s + b s^3 + c s^5; as a map of matrices its Lipschitz constant in the
Frobenius norm is max |p'| on [0, 1.21], which is below 4.2.  An error of relative size e in each step is therefore at most
e (4.2^5 - 1) / 3.2 = 408 e after five.  A step's own errors are roundings of 2^-24 (fp32 sums) and 2^-22 (the two-part operands) at a
handful of places (A, A A, P, the product, the stored X), independent from element to element: e = 2^-21 covers eight of
them.  So 408 * 2^-21 = 2e-4 of |out|_F, and for 16-bit results half a step of each element on top.  Long matrices take steps in
groups, which carry A along in place of X: A' = p A p passes an error of A on with at most a^2 = 11.9, X X^T of a step's X with
4.2^2.  (One lost part of an operand is 2^-12 per product, and shows as 1e-3 to 3e-3.)"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

A, B, C = 3.4445, -4.7750, 2.0315
HALF = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def _tolerance(steps):
    return (4.2 ** steps - 1) / 3.2 * 2.0 ** -21


@pytest.fixture(scope="module")
def torch():
    import torch
    import clusternet_amd as cn
    cn.init(0)
    return torch


def _exact(torch, G, steps=5):
    x = G.double()
    flip = x.shape[0] > x.shape[1]
    x = (x.T if flip else x).contiguous()
    x = x / (x.norm() + 1e-7)
    for _ in range(steps):
        a = x @ x.T.contiguous()
        x = A * x + (B * a + C * (a @ a)) @ x
    return x.T if flip else x


def _gradient(torch, rows, cols, seed, kind="noise"):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    g = torch.randn(rows, cols, generator=gen, device="cuda")
    if kind == "strong":  # a few directions far above the rest
        k = min(4, rows, cols)
        g = 0.02 * g + torch.randn(rows, k, generator=gen, device="cuda") @ torch.randn(k, cols, generator=gen, device="cuda")
    if kind == "identity":  # all entries that count alike, as all singular values
        g = torch.eye(rows, cols, device="cuda")
    if kind == "constant":
        g = torch.full_like(g, 0.37)
    if kind == "orthogonal":
        g = torch.linalg.qr((g if rows >= cols else g.T).contiguous()).Q
        g = (g if rows >= cols else g.T).contiguous()
    if kind == "repeated" and rows > 1:  # rank deficient
        g[rows - rows // 2:] = g[:rows // 2].clone()
    return g


def _close(torch, got, want, steps=5):
    name = str(got.dtype).split(".")[1]
    off = (got.double() - want).norm()
    allowed = _tolerance(steps) * want.norm() + (HALF[name] * want.norm() if name != "float32" else 0)
    assert bool(off <= allowed), (float(off), float(allowed))


SIZES = [(1, 1), (1, 7), (5, 1), (3, 4), (31, 33), (64, 64), (65, 257), (300, 10), (784, 1024), (1000, 129), (513, 512), (2048, 2048),
         (1500, 4100), (4500, 1030)]


@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("kind", ["noise", "strong", "repeated"])
def test_against_64_bits(torch, rows, cols, kind):
    import clusternet_amd as cn
    G = _gradient(torch, rows, cols, rows + cols, kind)
    out = cn.orthogonalize(G)
    _close(torch, out, _exact(torch, G))
    assert torch.equal(out, cn.orthogonalize(G))  # the same bits every time


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("rows,cols", [(1, 5), (100, 333), (784, 1024), (2100, 2050), (3000, 700)])
def test_16_bit_gradients(torch, dtype, rows, cols):
    import clusternet_amd as cn
    G = _gradient(torch, rows, cols, 3, "strong").to(getattr(torch, dtype))
    want = _exact(torch, G)
    out = cn.orthogonalize(G)
    assert out.dtype == G.dtype
    _close(torch, out, want)
    _close(torch, cn.orthogonalize(G, out=torch.empty(rows, cols, device="cuda")), want)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows,cols", [(17, 498), (300, 300), (100, 1700), (700, 2900), (4500, 1030)])
@pytest.mark.parametrize("kind", ["identity", "constant", "orthogonal"])
def test_equal_entries_and_singular_values(torch, rows, cols, dtype, kind):
    """Where roundings do not average out: the same in every entry, or passed on with the same slope.  In 32 bits of result too, so
    that nothing hides behind its rounding."""
    import clusternet_amd as cn
    G = _gradient(torch, rows, cols, 11, kind).to(getattr(torch, dtype))
    want = _exact(torch, G)
    _close(torch, cn.orthogonalize(G), want)
    _close(torch, cn.orthogonalize(G, out=torch.empty(rows, cols, device="cuda")), want)


@pytest.mark.parametrize("steps", [1, 2, 3, 8])
def test_numbers_of_steps(torch, steps):
    import clusternet_amd as cn
    G = _gradient(torch, 200, 150, 8)
    _close(torch, cn.orthogonalize(G, steps=steps), _exact(torch, G, steps), steps)


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 6, 7])
@pytest.mark.parametrize("rows,cols", [(700, 2900), (4500, 600)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_numbers_of_steps_of_long_matrices(torch, rows, cols, dtype, steps):
    import clusternet_amd as cn
    G = _gradient(torch, rows, cols, 9).to(getattr(torch, dtype))
    _close(torch, cn.orthogonalize(G, steps=steps, out=torch.empty(rows, cols, device="cuda")), _exact(torch, G, steps), steps)


def test_against_plain_32_bits(torch):
    """As far from the exact result as plain fp32 products, up to a factor of 1.5 and 1e-6, for well and badly conditioned
    gradients."""
    import clusternet_amd as cn
    for rows, cols in ((512, 512), (400, 1700)):
        for kind in ("noise", "strong", "repeated"):
            G = _gradient(torch, rows, cols, 21, kind)
            want = _exact(torch, G)
            x = G / (G.norm() + 1e-7)
            for _ in range(5):
                a = x @ x.T
                x = A * x + (B * a + C * (a @ a)) @ x
            plain = float((x.double() - want).norm() / want.norm())
            ours = float((cn.orthogonalize(G).double() - want).norm() / want.norm())
            assert ours <= max(1e-6, 1.5 * plain), (rows, cols, kind, ours, plain)


@pytest.mark.parametrize("rows,cols", [(3000, 16), (17, 500), (60, 3000), (120, 2500), (140, 5000), (1000, 4001)])
@pytest.mark.parametrize("kind", ["noise", "strong"])
def test_long_matrices_against_plain_32_bits(torch, rows, cols, kind):
    """Operands in two parts are rounded to 2^-23, twice fp32's 2^-24: at most twice as far, and 1e-6 for what is left to chance
    where both are that near."""
    import clusternet_amd as cn
    G = _gradient(torch, rows, cols, 31, kind)
    want = _exact(torch, G)
    x = (G if rows <= cols else G.T).contiguous()
    x = x / (x.norm() + 1e-7)
    for _ in range(5):
        a = x @ x.T.contiguous()
        x = A * x + (B * a + C * (a @ a)) @ x
    x = x if rows <= cols else x.T
    plain = float((x.double() - want).norm() / want.norm())
    ours = float((cn.orthogonalize(G).double() - want).norm() / want.norm())
    assert ours <= max(1e-6, 2 * plain), (ours, plain)


def test_scale_does_not_matter(torch):
    """Gradients of any finite size: powers of two change nothing until 1e-7 counts, and sums of squares do not overflow."""
    import clusternet_amd as cn
    G = _gradient(torch, 90, 210, 4)
    want = _exact(torch, G)
    for scale in (2.0 ** 100, 1e36, 2.0 ** -12):
        _close(torch, cn.orthogonalize(G * scale), want)
    tiny = G * 1e-9  # here 1e-7 is as large as the norm
    _close(torch, cn.orthogonalize(tiny), _exact(torch, tiny))


def test_zero_and_not_finite(torch):
    import clusternet_amd as cn
    assert not cn.orthogonalize(torch.zeros(40, 70, device="cuda")).any()
    for bad in (float("nan"), float("inf")):
        G = _gradient(torch, 40, 70, 1)
        G[7, 9] = bad
        assert bool(cn.orthogonalize(G).isnan().all())
    for dtype, rows, cols in ((torch.bfloat16, 40, 70), (torch.float16, 300, 2000), (torch.float32, 3000, 400), (torch.bfloat16, 3000, 400)):
        for bad in (float("nan"), float("inf"), -float("inf")):
            G = _gradient(torch, rows, cols, 2).to(dtype)
            G[rows - 1, cols - 1] = bad
            assert bool(cn.orthogonalize(G).isnan().all())
        assert not cn.orthogonalize(torch.zeros(rows, cols, device="cuda", dtype=dtype)).any()
    assert cn.orthogonalize(torch.empty(0, 5, device="cuda")).shape == (0, 5)
    assert cn.orthogonalize(torch.empty(5, 0, device="cuda")).shape == (5, 0)


def test_places(torch):
    """Parts of wider matrices, in place, and what surrounds the output stays."""
    import clusternet_amd as cn
    for rows, cols, off in ((130, 67, 1), (67, 130, 3), (64, 64, 0)):
        wide = _gradient(torch, rows + 2, cols + 9, 17)
        G = wide[1:rows + 1, off:off + cols]
        want = _exact(torch, G)
        back = torch.full((rows + 3, cols + 11), 7.0, device="cuda")
        out = back[2:rows + 2, off + 1:off + 1 + cols]
        cn.orthogonalize(G, out=out)
        _close(torch, out, want)
        keep = torch.ones_like(back, dtype=torch.bool)
        keep[2:rows + 2, off + 1:off + 1 + cols] = False
        assert bool((back[keep] == 7.0).all())
        before = wide.clone()
        assert cn.orthogonalize(G, out=G) is G
        assert torch.equal(G, out)
        wide[1:rows + 1, off:off + cols] = before[1:rows + 1, off:off + cols]
        assert torch.equal(wide, before)


@pytest.mark.parametrize("rows,cols", [(1, 3), (100, 60), (784, 1024), (2050, 2049)])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_update(torch, rows, cols, dtype, nesterov):
    """Momentum bit for bit (a product and a sum, rounded each); weights to the direction's tolerance plus their own roundings."""
    import clusternet_amd as cn
    mu, rate, decay = 0.95, 0.02, 0.1
    f = np.float32
    grad = _gradient(torch, rows, cols, 5, "strong").to(getattr(torch, dtype))
    mom, w = _gradient(torch, rows, cols, 6), 0.1 * _gradient(torch, rows, cols, 7)
    want_mom = mom * float(f(mu)) + grad.float()
    u = grad.float() + want_mom * float(f(mu)) if nesterov else want_mom
    keep = float(f(1) - f(rate) * f(decay))
    o = _exact(torch, u)
    want_w = keep * w.double() - float(f(rate)) * o
    got_mom, got_w = cn.muon_update(mom, grad, w, mu, rate, nesterov=nesterov, weight_decay=decay)
    assert got_mom is mom and got_w is w
    assert torch.equal(mom, want_mom)
    off = (w.double() - want_w).norm()
    assert bool(off <= rate * _tolerance(5) * o.norm() + 4 * 2.0 ** -24 * (want_w.norm() + rate * o.norm())), float(off)


def test_muon_in_strided_places(torch):
    import clusternet_amd as cn
    wides = [_gradient(torch, 70, 50, s) for s in (1, 2, 3)]
    keep = [x.clone() for x in wides]
    mom, grad, w = (x[3:64, 5 + i:46 + i] for i, x in enumerate(wides))
    alone = [x.clone().contiguous() for x in (mom, grad, w)]
    cn.muon_update(mom, grad, w, 0.9, 0.1)
    cn.muon_update(*alone, 0.9, 0.1)
    assert torch.equal(mom, alone[0]) and torch.equal(w, alone[2])
    for i, (x, k) in enumerate(zip(wides, keep)):
        x[3:64, 5 + i:46 + i] = k[3:64, 5 + i:46 + i]
        assert torch.equal(x, k)


def test_in_graphs_and_on_other_streams(torch):
    """Two captured graphs with eager work between their replays and a call on a side stream: the eager bits every time."""
    import clusternet_amd as cn
    sets = []
    for rows, cols in ((200, 333), (600, 130)):
        G = _gradient(torch, rows, cols, rows)
        cn.orthogonalize(G)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = cn.orthogonalize(G)
        sets.append((G, graph, got))
    side = torch.cuda.Stream()
    for k in range(4):
        for G, graph, got in sets:
            G.copy_(_gradient(torch, G.shape[0], G.shape[1], 100 + k))
            want = cn.orthogonalize(G)
            with torch.cuda.stream(side):
                side.wait_stream(torch.cuda.default_stream())
                beside = cn.orthogonalize(G)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want) and torch.equal(beside, want)
