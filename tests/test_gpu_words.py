"""A maxout net that reads words, as a run: lookup, forward, backward, the gradient of the table, orthogonalised updates, then
answers from weights in 4 bits.

The 64-bit reference carries a bound with each number (`Bounded`): what the device may be off by if its inputs are off by their
bounds and each of its sums of K terms by K + 8 whole fp32 steps (2^-23) of the sum of their magnitudes, so no tolerance is chosen.
Gradients follow the device's winners (the branch taken where two pool members are equal within rounding); the formula's
gradient itself is held against differences of the 64-bit loss on the same branch."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -23


@pytest.fixture(scope="module")
def torch():
    import torch
    import clusternet_amd as cn
    cn.init(0)
    return torch


class Bounded:
    def __init__(self, v, e=0.0):
        self.v = np.asarray(v, np.float64)
        self.e = np.broadcast_to(np.asarray(e, np.float64), self.v.shape)

    @property
    def T(self):
        return Bounded(self.v.T, self.e.T)

    def __matmul__(self, o):
        a, b = np.abs(self.v), np.abs(o.v)
        top = (a + self.e) @ (b + o.e)
        return Bounded(self.v @ o.v, top - a @ b + (self.v.shape[1] + 8) * U * top)

    def rounded(self):  # one more operation of the device
        return Bounded(self.v, self.e + U * (np.abs(self.v) + self.e))

    def __add__(self, o):
        return Bounded(self.v + o.v, self.e + o.e).rounded()

    def __sub__(self, o):
        return Bounded(self.v - o.v, self.e + o.e).rounded()

    def times(self, s):
        return Bounded(self.v * s, self.e * abs(s)).rounded()

    def take(self, columns):
        rows = np.arange(len(self.v))[:, None]
        return Bounded(self.v[rows, columns], self.e[rows, columns])

    def expand(self, columns, width):
        v, e = np.zeros((len(self.v), width)), np.zeros((len(self.v), width))
        rows = np.arange(len(self.v))[:, None]
        v[rows, columns], e[rows, columns] = self.v, self.e
        return Bounded(v, e)

    def pool_max(self, pool):
        shape = (len(self.v), -1, pool)
        return Bounded(self.v.reshape(shape).max(2), self.e.reshape(shape).max(2))

    def softmax(self):
        """exp(z - max) / sum: z is off by e and one rounding of the difference to the largest, exp by 4 steps, the sum by a step
        per term, the quotient by 2."""
        z = self.v - self.v.max(1, keepdims=True)
        p = np.exp(z)
        p /= p.sum(1, keepdims=True)
        spread = 2 * self.e.max(1, keepdims=True) + U * np.abs(z).max(1, keepdims=True)
        return Bounded(p, p * (np.expm1(2 * spread) + (z.shape[1] + 16) * U))

    def holds(self, got):
        got = np.asarray(got.double().cpu().numpy())
        assert got.shape == self.v.shape and np.isfinite(got).all()
        # 2^-120: far above what subnormals can lose, far below every number here
        assert (np.abs(got - self.v) <= self.e + 2.0 ** -120).all(), (np.abs(got - self.v) - self.e).max()


def _net(torch, batch, window, rows, D, H, O, seed, token_type="int64"):
    g = torch.Generator(device="cuda").manual_seed(seed)
    u = lambda r, c: (torch.rand((r, c), device="cuda", generator=g) * 2 - 1) * (6.0 / (r + c)) ** 0.5  # noqa: E731
    table = torch.randn((rows, D), device="cuda", generator=g)
    params = (u(window * D, 2 * H), torch.randn(2 * H, device="cuda", generator=g) * 0.1, u(H, 2 * H),
              torch.randn(2 * H, device="cuda", generator=g) * 0.1, u(H, O), torch.randn(O, device="cuda", generator=g) * 0.1)
    tokens = torch.randint(0, rows, (batch, window), device="cuda", generator=g).to(getattr(torch, token_type))
    onehot = torch.nn.functional.one_hot(torch.randint(0, O, (batch,), device="cuda", generator=g), O).float()
    return table, params, tokens, onehot


def _bounded(t):
    return Bounded(t.double().cpu().numpy())


def _rows(table, tokens, scale):
    """The lookup of 64-bit rows; zeros for a token outside the table."""
    t = tokens.cpu().numpy()
    inside = (t >= 0) & (t < len(table))
    return (scale * table[np.where(inside, t, 0)] * inside[..., None]).reshape(len(t), -1)


def _reference(table, tokens, scale, params, onehot, columns, pool=2):
    """(p, gradients of the three matrices, e0, gradient of the table), 64 bits with bounds, on the branch `columns`."""
    W1, b1, W2, b2, W3, b3 = (_bounded(t) for t in params)
    y, t = _bounded(onehot), tokens.cpu().numpy()
    X = Bounded(_rows(table.double().cpu().numpy(), tokens, scale)).rounded()
    z1 = X @ W1 + b1
    h1 = z1.take(columns[0])
    z2 = h1 @ W2 + b2
    h2 = z2.take(columns[1])
    for z, h in ((z1, h1), (z2, h2)):  # the device took a winner, within rounding
        assert (z.pool_max(pool).v - h.v <= 2 * z.pool_max(pool).e).all()
    p = (h2 @ W3 + b3).softmax()
    e3 = p - y
    e2 = (e3 @ W3.T).expand(columns[1], z2.v.shape[1])
    e1 = (e2 @ W2.T).expand(columns[0], z1.v.shape[1])
    e0 = e1 @ W1.T
    D = table.shape[1]
    v, e, top, n = (np.zeros(table.shape) for _ in range(4))
    for at, value in ((v, e0.v), (e, e0.e), (top, np.abs(e0.v) + e0.e), (n, np.ones_like(e0.v))):
        flat, inside = t.reshape(-1), (t.reshape(-1) >= 0) & (t.reshape(-1) < len(table))
        np.add.at(at, flat[inside], value.reshape(-1, D)[inside])
    dE = Bounded(v, e + (n + 8) * U * top).times(scale)
    return p, (X.T @ e1, h1.T @ e2, h2.T @ e3), e0, dE


SHAPES = [(1, 1, 3, 1, 4, 2), (64, 11, 500, 24, 64, 10), (33, 5, 7, 13, 50, 17), (128, 11, 1000, 60, 128, 30)]


@pytest.mark.parametrize("batch,window,rows,D,H,O", SHAPES)
@pytest.mark.parametrize("token_type", ["int32", "int64"])
def test_forward_and_gradients(torch, batch, window, rows, D, H, O, token_type):
    from clusternet_amd import maxout_step as ms
    scale = 0.75
    table, params, tokens, onehot = _net(torch, batch, window, rows, D, H, O, batch + D, token_type)
    if tokens.numel() > 3:
        tokens.view(-1)[-2:] = torch.tensor([-1, rows], device="cuda")  # padding at the end of the last window
    X = ms.token_input(table, tokens, scale)
    p, cache = ms.forward(X, params)
    columns = [cache[i].cpu().numpy().astype(np.int64) for i in (1, 3)]
    want_p, want_g, want_e0, want_dE = _reference(table, tokens, scale, params, onehot, columns)
    want_p.holds(p)
    got = ms.backward(X, onehot, params, p, cache)
    for w, g in zip(want_g + (want_e0,), got):
        w.holds(g)
    before = table.clone()
    ms.table_update(X, got[3], 1.0)
    named = torch.zeros(rows, dtype=torch.bool, device="cuda")
    named[tokens[(tokens >= 0) & (tokens < rows)].long()] = True
    assert torch.equal(table[~named], before[~named])
    change = Bounded(before.double().cpu().numpy() - want_dE.v, want_dE.e).rounded()
    change.holds(table)


def test_formula_against_differences(torch):
    """The reference's own gradients: central differences of the 64-bit loss along random directions, on the same branch.  With
    steps of 1e-4 along directions of length one a difference is off by about 1e-8 of the third derivative."""
    from clusternet_amd import maxout_step as ms
    table, params, tokens, onehot = _net(torch, 20, 4, 15, 6, 16, 5, 1)
    X = ms.token_input(table, tokens)
    _, cache = ms.forward(X, params)
    columns = [cache[i].cpu().numpy().astype(np.int64) for i in (1, 3)]
    _, grads, _, dE = _reference(table, tokens, 1.0, params, onehot, columns)
    rows = np.arange(20)[:, None]
    b = [params[i].double().cpu().numpy() for i in (1, 3, 5)]
    y = onehot.double().cpu().numpy()

    def loss(E, W1, W2, W3):
        h1 = (_rows(E, tokens, 1.0) @ W1 + b[0])[rows, columns[0]]
        h2 = (h1 @ W2 + b[1])[rows, columns[1]]
        z = h2 @ W3 + b[2]
        return (np.log(np.exp(z).sum(1)) - (z * y).sum(1)).sum()

    at = [table.double().cpu().numpy()] + [params[i].double().cpu().numpy() for i in (0, 2, 4)]
    rng = np.random.default_rng(2)
    for i, g in enumerate([dE.v] + [g.v for g in grads]):
        d = rng.normal(size=at[i].shape)
        d /= np.linalg.norm(d)
        up, down = list(at), list(at)
        up[i], down[i] = at[i] + 1e-4 * d, at[i] - 1e-4 * d
        slope = (loss(*up) - loss(*down)) / 2e-4
        assert abs(slope - (g * d).sum()) <= 1e-6 * np.linalg.norm(g)


def _state(torch, seed=5):
    table, params, tokens, onehot = _net(torch, 128, 11, 700, 60, 128, 20, seed)
    return table, params, tokens, onehot, [torch.zeros_like(params[0]), torch.zeros_like(params[2])]


def test_step_is_its_parts(torch):
    """token_step, to the bit: forward, backward, two orthogonalised updates, the 8-bit update and the table's."""
    import clusternet_amd as cn
    from clusternet_amd import maxout_step as ms
    table, params, tokens, onehot, momenta = _state(torch)
    table2, params2, momenta2 = table.clone(), [t.clone() for t in params], [m.clone() for m in momenta]
    for _ in range(3):
        p = ms.token_step(ms.token_input(table, tokens), onehot, params, momenta, 0.02, 0.1)
        X = ms.token_input(table2, tokens)
        p2, cache = ms.forward(X, params2)
        g1, g2, g3, e0 = ms.backward(X, onehot, params2, p2, cache)
        cn.muon_update(momenta2[0], g1, params2[0], 0.95, 0.02)
        cn.muon_update(momenta2[1], g2, params2[2], 0.95, 0.02)
        ms.coded_update(params2[4], g3, 0.01)
        ms.table_update(X, e0, 0.1)
        assert torch.equal(p, p2) and torch.equal(table, table2)
        for a, b in zip(list(params) + momenta, params2 + momenta2):
            assert torch.equal(a, b) and torch.isfinite(a).all()


def test_captured_step(torch):
    """The step in a graph: three replays, eager work between them, give the bits of three eager steps."""
    from clusternet_amd import maxout_step as ms
    table, params, tokens, onehot, momenta = _state(torch, 6)
    copies = [t.clone() for t in [table, *params, *momenta]]
    table2, params2, momenta2 = copies[0], copies[1:7], copies[7:]
    run = lambda: ms.token_step(ms.token_input(table2, tokens), onehot, params2, momenta2, 0.02, 0.1)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    for t, start in zip([table2, *params2, *momenta2], [table, *params, *momenta]):
        t.copy_(start)
    with torch.cuda.graph(graph):
        p2 = run()
    for _ in range(3):
        p = ms.token_step(ms.token_input(table, tokens), onehot, params, momenta, 0.02, 0.1)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(p, p2)
        for a, b in zip([table, *params, *momenta], [table2, *params2, *momenta2]):
            assert torch.equal(a, b)


@pytest.mark.parametrize("batch", [1, 3, 40])
@pytest.mark.parametrize("group,zero_points", [(32, False), (64, True), (128, False), (128, True)])
def test_answers_from_4_bits(torch, batch, group, zero_points):
    """`answer` against the 64-bit net of the weights that the codes stand for.  The products with 4-bit weights sum a (16 + q) and
    a apart (terms up to 62 |a| s in place of |a (q - z)| s), so their bound is K + 8 steps of that sum."""
    from clusternet_amd import maxout_step as ms
    import clusternet_amd as cn
    table, params, tokens, onehot = _net(torch, batch, 11, 300, 25, 96, 20, 7)
    params4 = ms.quantize_params(params, group, zero_points)
    X = ms.token_input(table, tokens)
    p = ms.answer(X, params4)
    assert torch.equal(p, ms.answer(X.X, params4))

    def product(h, w4):
        w = _bounded(cn.dequantize_4bit(w4))
        s = np.repeat(w4.scales.double().cpu().numpy(), group, 0)[:w4.inner]
        out = h @ w
        return Bounded(out.v, out.e + (w4.inner + 8) * U * 62 * ((np.abs(h.v) + h.e) @ s) + U * (np.abs(h.v) + h.e) @ np.abs(w.v))

    h = Bounded(_rows(table.double().cpu().numpy(), tokens, 1.0))
    for i in (0, 2):
        h = (product(h, params4[i]) + _bounded(params[i + 1])).pool_max(2)
    (product(h, params4[4]) + _bounded(params[5])).softmax().holds(p)


def test_words_are_refused_in_the_wrong_shape(torch):
    from clusternet_amd import maxout_step as ms
    table, params, tokens, _ = _net(torch, 4, 3, 10, 4, 8, 3, 9)
    with pytest.raises(ValueError):
        ms.token_input(table, tokens.view(-1))
    with pytest.raises(TypeError):
        ms.token_input(table, tokens.float())
