"""cn_gemm_w4 on fp32 rows beside a plain fp32 product of the decoded weights, both against 64 bits.

Products are exact (three parts of a row's number of 8 bits each, whole numbers of 4 bits), so what is rounded are the sums: three per
32 numbers of K, one for each part, where a plain product has one at most that often in the largest instruction there is.  Rounding
errors of that many independent sums are sqrt(3) < 2 times as far off, root mean square over the columns, whatever the rows
look like; the scale's own rounding is the decoded weights' too.  1e-7 of the largest result, two of fp32's half steps, is left to
chance where a plain product happens to be exact."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    import clusternet_amd as cn
    cn.init(0)
    return torch


def _rows(torch, kind, M, K, gen):
    x = torch.randn(M, K, 2, device="cuda", generator=gen)
    if kind == "normal":
        return x[..., 0].contiguous()
    if kind == "maxout":  # what a maxout layer hands on
        return x.amax(-1)
    if kind == "sigmoid":
        return x[..., 0].sigmoid()
    return 1 + 1e-3 * x[..., 0]  # nearly equal


@pytest.mark.parametrize("kind", ["normal", "maxout", "sigmoid", "near one"])
@pytest.mark.parametrize("M,K,N", [(1, 4096, 1000), (13, 5000, 1999), (5, 2051, 8300), (40, 4096, 600), (64, 1000, 8300)])
@pytest.mark.parametrize("group,zero_points", [(32, True), (64, False), (128, True), (128, False)])
def test_rows_with_a_mean(torch, kind, M, K, N, group, zero_points):
    import clusternet_amd as cn
    gen = torch.Generator(device="cuda").manual_seed(M + K)
    w4 = cn.quantize_4bit(0.02 * torch.randn(K, N, device="cuda", generator=gen), group, zero_points)
    x = _rows(torch, kind, M, K, gen)
    w = cn.dequantize_4bit(w4)
    want = x.double() @ w.double()
    off = lambda y: float((y.double() - want).square().mean().sqrt())  # noqa: E731
    ours, plain = off(cn.gemm_w4(x, w4)), off(x @ w)
    assert ours <= max(2 * plain, 1e-7 * float(want.abs().max())), (ours / plain, ours / float(want.abs().max()))
