"""cn_orthogonalize beside the same steps in plain fp32, both against 64 bits: 16-bit gradients, which are used as they are, with 32
bits of result, and more than the usual steps.

A number in two fp16 parts is off by up to 2^-23 of its power of two, one in fp32 by 2^-24: at most twice as far, and 1e-6 for what is
left to chance where both are that near."""
import pytest

pytestmark = pytest.mark.gpu

A, B, C = 3.4445, -4.7750, 2.0315


@pytest.fixture(scope="module")
def torch():
    import torch
    import clusternet_amd as cn
    cn.init(0)
    return torch


def _steps(G, steps=5):
    x = G.T.contiguous() if G.shape[0] > G.shape[1] else G
    x = x / (x.double().norm().to(x.dtype) + 1e-7)
    for _ in range(steps):
        a = x @ x.T.contiguous()
        x = A * x + (B * a + C * (a @ a)) @ x
    return x.T if G.shape[0] > G.shape[1] else x


def _gradient(torch, rows, cols, kind, gen):
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    G = torch.zeros(rows, cols, device="cuda")
    if kind == "one row":
        G[rows // 2] = r(cols)
    elif kind == "two rows":
        G[1:3] = r(2, cols)
    elif kind == "sixteen rows":
        G[::rows // 16][:16] = r(16, cols)
    elif kind == "equal rows":
        G[3:5] = r(1, cols)
    elif kind == "one column":
        G[:, 5] = r(rows)
    elif kind == "half of the rows":
        G[::2] = r(rows, cols)[::2]
    elif kind == "one direction":
        G = r(rows, 1) @ r(1, cols)
    elif kind == "strong":
        G = 0.02 * r(rows, cols) + r(rows, 4) @ r(4, cols)
    else:
        G = r(rows, cols)
    return G


KINDS = ["one row", "two rows", "sixteen rows", "equal rows", "one column", "half of the rows", "one direction", "noise"]


@pytest.mark.parametrize("rows,cols", [(140, 5000), (256, 6000), (700, 2900), (2900, 700), (100, 900), (300, 300)])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_few_rows_and_directions(torch, rows, cols, kind, dtype):
    """Where few rows, columns or directions carry the gradient, roundings do not average out: their root mean square over
    several gradients.  A number in two fp16 parts is off by up to 2^-23 of its power of two, one in fp32 by 2^-24: 1.15 and 0.58 times
    2^-24, root mean square.  A product leaves out lo lo, two errors of up to 2^-11: 1.33 times 2^-24 where a sum has one term,
    less where it has more.  A step rounds A, P and X and computes three products from them: sqrt(3 * 1.15^2 + 3 * 1.33^2)
    against sqrt(3 * 0.58^2), so no more than 3.05 times as far as plain fp32."""
    import clusternet_amd as cn
    gen = torch.Generator(device="cuda").manual_seed(rows)
    ours = plain = 0.0
    for _ in range(6):
        G = _gradient(torch, rows, cols, kind, gen).to(getattr(torch, dtype))
        want = _steps(G.double())
        far = lambda x: float((x.double() - want).norm() / want.norm()) ** 2 / 6  # noqa: E731
        ours += far(cn.orthogonalize(G, out=torch.empty(rows, cols, device="cuda")))
        plain += far(_steps(G.float()))
    assert ours ** 0.5 <= 3.05 * plain ** 0.5, (ours ** 0.5, plain ** 0.5, (ours / plain) ** 0.5)


@pytest.mark.parametrize("rows,cols", [(100, 333), (784, 1024), (2100, 2050), (3000, 700), (700, 2900)])
@pytest.mark.parametrize("kind", ["noise", "strong"])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("steps", [1, 2, 5])
def test_16_bit_gradients_lose_nothing_more(torch, rows, cols, kind, dtype, steps):
    """Used as they are, with the power of two of their scale: in 32 bits of result as near as fp32 gradients."""
    import clusternet_amd as cn
    G = _gradient(torch, rows, cols, kind, torch.Generator(device="cuda").manual_seed(7)).to(getattr(torch, dtype))
    want = _steps(G.double(), steps)
    far = lambda x: float((x.double() - want).norm() / want.norm())  # noqa: E731
    ours, plain = far(cn.orthogonalize(G, steps, out=torch.empty(rows, cols, device="cuda"))), far(_steps(G.float(), steps))
    assert ours <= max(1e-6, 2 * plain), (ours, plain)


@pytest.mark.parametrize("rows,cols", [(200, 150), (700, 2900), (4500, 600)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("steps", [6, 7, 8, 12])
def test_many_steps(torch, rows, cols, dtype, steps):
    """What a step passes on grows alike in both."""
    import clusternet_amd as cn
    G = _gradient(torch, rows, cols, "noise", torch.Generator(device="cuda").manual_seed(9)).to(getattr(torch, dtype))
    want = _steps(G.double(), steps)
    far = lambda x: float((x.double() - want).norm() / want.norm())  # noqa: E731
    ours, plain = far(cn.orthogonalize(G, steps, out=torch.empty(rows, cols, device="cuda"))), far(_steps(G.float(), steps))
    assert ours <= max(1e-6, 2 * plain), (ours, plain)


@pytest.mark.parametrize("rows,cols", [(4500, 600), (600, 4500), (700, 2900), (400, 400), (2048, 2048), (784, 1024)])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_every_row_of_two_steps(torch, rows, cols, dtype):
    """A single wrong element of X X^T is a multiple of one row in another.  Of noise, X X^T counts little in two steps: what is rounded
    is the stored X (0.58 of 2^-23, root mean square over a row), two sums (2^-24 each) and three factors (2^-24 each): less
    than 4 * 2^-23 of every row."""
    import clusternet_amd as cn
    for seed in (1, 2, 3, 9):
        G = _gradient(torch, rows, cols, "noise", torch.Generator(device="cuda").manual_seed(seed)).to(getattr(torch, dtype))
        want = _steps(G.double(), 2)
        off = cn.orthogonalize(G, 2, out=torch.empty(rows, cols, device="cuda")).double() - want
        along = 0 if rows > cols else 1
        worst = float((off.norm(dim=along) / want.norm(dim=along)).max())
        assert worst <= 4 * 2.0 ** -23, worst
