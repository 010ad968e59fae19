"""One TokenInput over several steps: the table moves under it, and every pass takes the rows as they are then."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    import clusternet_amd as cn
    cn.init(0)
    return torch


def _net(torch, seed, batch=32, window=5, rows=60, D=12, H=32, O=7):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: 0.3 * torch.randn(s, device="cuda", generator=g)  # noqa: E731
    params = [r(window * D, 2 * H), r(2 * H), r(H, 2 * H), r(2 * H), r(H, O), r(O)]
    tokens = torch.randint(0, rows, (batch, window), device="cuda", generator=g)
    onehot = torch.nn.functional.one_hot(torch.randint(0, O, (batch,), device="cuda", generator=g), O).float()
    return r(rows, D), params, [torch.zeros_like(params[0]), torch.zeros_like(params[2])], tokens, onehot


def test_steps_and_answers_on_one_input(torch):
    """To the bit what a fresh input per step gives, table, weights and answers."""
    from clusternet_amd import maxout_step as ms
    table, params, momenta, tokens, onehot = _net(torch, 1)
    table2, params2, momenta2, _, _ = _net(torch, 1)
    X = ms.token_input(table, tokens, 0.5)
    for _ in range(3):
        p = ms.token_step(X, onehot, params, momenta, 0.02, 0.5)
        assert torch.equal(p, ms.token_step(ms.token_input(table2, tokens, 0.5), onehot, params2, momenta2, 0.02, 0.5))
        for a, b in zip([table, *params, *momenta], [table2, *params2, *momenta2]):
            assert torch.equal(a, b)
        params4 = ms.quantize_params(params)
        assert torch.equal(ms.answer(X, params4), ms.answer(ms.token_input(table, tokens, 0.5), params4))
        assert torch.equal(ms.forward(X, params)[0], ms.forward(ms.token_input(table, tokens, 0.5), params)[0])


def test_new_words_in_the_same_place(torch):
    from clusternet_amd import maxout_step as ms
    table, params, _, tokens, _ = _net(torch, 2)
    X = ms.token_input(table, tokens)
    ms.forward(X, params)
    tokens.copy_(tokens.flip(0).clone())
    assert torch.equal(ms.forward(X, params)[0], ms.forward(table[tokens].view(len(tokens), -1), params)[0])


def test_gradients_are_those_of_their_own_forward(torch):
    """The table moves between a forward pass and its backward pass: the gradients stay those of the rows that were looked up."""
    from clusternet_amd import maxout_step as ms
    table, params, _, tokens, onehot = _net(torch, 3)
    X = ms.token_input(table, tokens)
    p, cache = ms.forward(X, params)
    want = ms.backward(X, onehot, params, p, cache)
    table.mul_(-2.0)
    for a, b in zip(want, ms.backward(X, onehot, params, p, cache)):
        assert torch.equal(a, b)


def test_one_captured_input(torch):
    """A graph of a step on an input made outside of it: each replay looks up what the replay before left in the table."""
    from clusternet_amd import maxout_step as ms
    table, params, momenta, tokens, onehot = _net(torch, 4)
    table2, params2, momenta2, _, _ = _net(torch, 4)
    X = ms.token_input(table2, tokens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ms.token_step(X, onehot, params2, momenta2, 0.02, 0.5)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p2 = ms.token_step(X, onehot, params2, momenta2, 0.02, 0.5)
    ms.token_step(ms.token_input(table, tokens), onehot, params, momenta, 0.02, 0.5)
    for _ in range(3):
        p = ms.token_step(ms.token_input(table, tokens), onehot, params, momenta, 0.02, 0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(p, p2)
        for a, b in zip([table, *params, *momenta], [table2, *params2, *momenta2]):
            assert torch.equal(a, b)


def test_answers_with_biases_of_any_shape(torch):
    from clusternet_amd import maxout_step as ms
    table, params, _, tokens, _ = _net(torch, 5)
    X = ms.token_input(table, tokens)
    want = ms.answer(X, ms.quantize_params(params))
    for shape in ((1, -1), (-1, 1)):
        shaped = [t if i % 2 == 0 else t.view(shape) for i, t in enumerate(params)]
        assert torch.equal(ms.forward(X, shaped)[0], ms.forward(X, params)[0])
        assert torch.equal(ms.answer(X, ms.quantize_params(shaped)), want)
