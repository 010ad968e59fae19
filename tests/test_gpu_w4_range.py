"""cn_gemm_w4 over the whole range of its operands, against 64 bits.

The bound is a count of roundings: a group's sums of at most 128 terms, groups and wavefronts that add up to K / group + 8 further
ones, a whole step (2^-23) each, of terms no larger than 62 |a| s.  Numbers of 2^-126 and less may lose what is below 2^-149 times the
2^13 that sums are kept below their values: 2^-136 s a term, and 2^-126 in the result itself (fp16: half of its smallest step, 2^-25).
What has to be finite: results whose sum of |a w| is, since partial sums are no larger."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HALF = {"float32": 0.0, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
LEAST = {"float32": 2.0 ** -126, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -126}


@pytest.fixture(scope="module")
def torch():
    import torch
    import clusternet_amd as cn
    cn.init(0)
    return torch


def _holds(torch, a, w4):
    import clusternet_amd as cn
    out = cn.gemm_w4(a, w4).double().cpu().numpy()
    ad = a.double().cpu().numpy()
    K, N, group = w4.inner, w4.outer, w4.group
    s = np.repeat(w4.scales.double().cpu().numpy(), group, 0)[:K]
    words = w4.codes.cpu().numpy().view(np.uint32)
    l, t, i = np.meshgrid(np.arange(64), np.arange(4), np.arange(8), indexing="ij")
    q = np.zeros((words.shape[1] * 128, words.shape[0] * 16))
    for x in range(words.shape[0]):
        for b in range(words.shape[1]):
            q[128 * b + 32 * t + 8 * (l // 16) + i, 16 * x + l % 16] = (words[x, b, l, t] >> (4 * i).astype(np.uint32)) & 15
    z = 8.0 if w4.zeros is None else np.repeat(w4.zeros.cpu().numpy().astype(np.float64), group, 0)[:K]
    w = (q[:K, :N] - z) * s
    want, top = ad @ w, np.abs(ad) @ np.abs(w)
    name = str(a.dtype).split(".")[1]
    bound = (128 + K / group + 16) * 2.0 ** -23 * 62 * (np.abs(ad) @ s) + 2.0 ** -136 * K * s.max(0) + LEAST[name]
    bound = bound * (1 + HALF[name]) + HALF[name] * np.abs(want)
    largest = float(torch.finfo(a.dtype).max)
    finite = top + bound < float(torch.finfo(a.dtype).max)
    assert np.isfinite(out[finite]).all()
    off = np.abs(out[finite] - want[finite])
    assert (off <= bound[finite]).all(), float((off - bound[finite]).max())
    return out, want


def _weights(torch, K, N, group, zero_points, size, seed=1):
    import clusternet_amd as cn
    rng = np.random.default_rng(seed)
    return cn.quantize_4bit(torch.from_numpy((size * rng.uniform(-1, 1, (K, N))).astype(np.float32)).cuda(), group, zero_points)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("group,zero_points", [(32, True), (64, False), (128, True), (128, False)])
@pytest.mark.parametrize("M", [1, 20])
@pytest.mark.parametrize("K,N", [(256, 33), (300, 17)])
def test_large_rows(torch, dtype, group, zero_points, M, K, N):
    """Rows of one sign and of both, up to the largest number, where the results are finite by far."""
    w4 = _weights(torch, K, N, group, zero_points, 1e-4)
    rng = np.random.default_rng(2)
    for size in (1e33, 8e34, 1e37, 3e38, 3.38e38):
        for signs in (np.ones((M, K)), np.sign(rng.normal(size=(M, K)))):
            a = torch.from_numpy((size * signs * rng.uniform(0.99, 1, (M, K))).astype(np.float32)).cuda().to(getattr(torch, dtype))
            out, want = _holds(torch, a, w4)
            assert np.isfinite(out).all()


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("group,zero_points", [(32, True), (128, False)])
@pytest.mark.parametrize("size,rows", [(1e36, 1e-3), (3e38, 1e-6), (3e38, 1.0), (1e-36, 1.0), (1e-42, 1e4), (1.0, 1e-36), (1e-3, 1e-42), (1e-30, 1e30)])
def test_large_and_small_scales_and_rows(torch, dtype, group, zero_points, size, rows):
    w4 = _weights(torch, 200, 40, group, zero_points, size)
    rng = np.random.default_rng(3)
    a = torch.from_numpy((rows * rng.uniform(-1, 1, (5, 200))).astype(np.float32)).cuda().to(getattr(torch, dtype))
    if bool(a.isfinite().all()):  # (fp16 holds no 1e30)
        _holds(torch, a, w4)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("group,zero_points", [(32, True), (64, False), (128, False)])
@pytest.mark.parametrize("M", [4, 20])
def test_rows_that_are_not_finite(torch, dtype, group, zero_points, M):
    """NaN all along them, whatever the weights, and nothing of it in other rows."""
    import clusternet_amd as cn
    w4 = _weights(torch, 200, 40, group, zero_points, 0.1)
    a = torch.randn(M, 200, device="cuda", generator=torch.Generator(device="cuda").manual_seed(4)).to(getattr(torch, dtype))
    want = cn.gemm_w4(a, w4)
    a[1, 0], a[2, 199], a[3, 64] = float("nan"), float("inf"), -float("inf")
    out = cn.gemm_w4(a, w4)
    rest = [0, *range(4, M)]
    assert bool(out[1:4].isnan().all()) and torch.equal(out[rest], want[rest])
