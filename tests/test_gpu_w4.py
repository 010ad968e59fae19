"""cn_quantize_4bit, cn_dequantize_4bit and cn_gemm_w4 through the binding.

Quantisation is held to its definition exactly: scales rounded once, codes decided in 64 bits with halves to even.  Products on
whole numbers with power-of-two scales are exact in any order and held bit for bit.  Otherwise: a group's two sums (of
a (16 + q), 16 + q <= 31, and of a) have at most 128 exact terms, the second is multiplied by at most 31, and groups and
wavefronts add up to K / group + 8 further terms; a matrix instruction's additions are taken to be off by a whole step, 2^-23.
So |out - exact| <= (128 + K / group + 16) 2^-23 * 62 sum |a| s, and half a step of the result for 16 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HALF = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


@pytest.fixture(scope="module")
def torch():
    import torch
    import clusternet_amd as cn
    cn.init(0)
    return torch


def _codes(codes, K, N):
    """The numbers 0 .. 15 of the stored form, K x N, by its definition, and whether the padding holds 0."""
    words = codes.cpu().numpy().view(np.uint32)
    nt, kb = words.shape[:2]
    a, b, l, t, i = np.meshgrid(np.arange(nt), np.arange(kb), np.arange(64), np.arange(4), np.arange(8), indexing="ij")
    q = (words[a, b, l, t] >> (4 * i)) & 15
    full = np.zeros((kb * 128, nt * 16), np.int64)
    full[128 * b + 32 * t + 8 * (l // 16) + i, 16 * a + l % 16] = q
    return full[:K, :N], not (full[K:].any() or full[:, N:].any())


def _stored(q):
    K, N = q.shape
    nt, kb = -(-N // 16), -(-K // 128)
    full = np.zeros((kb * 128, nt * 16), np.uint32)
    full[:K, :N] = q
    a, b, l, t, i = np.meshgrid(np.arange(nt), np.arange(kb), np.arange(64), np.arange(4), np.arange(8), indexing="ij")
    return np.bitwise_or.reduce(full[128 * b + 32 * t + 8 * (l // 16) + i, 16 * a + l % 16] << (4 * i).astype(np.uint32), axis=-1).view(np.int32)


def _definition(w, group, zero_points):
    """(q, scales, zeros) of float64 weights."""
    K, N = w.shape
    groups = -(-K // group)
    scales, zeros, q = np.zeros((groups, N), np.float32), np.full((groups, N), 8, np.int64), np.zeros((K, N), np.int64)
    with np.errstate(all="ignore"):
        for g in range(groups):
            part = w[g * group:(g + 1) * group]
            if zero_points:
                hi, lo = np.maximum(part.max(0), 0), np.minimum(part.min(0), 0)
                s = ((hi - lo) / 15).astype(np.float32)
                z = np.where(s > 0, np.rint(-lo / s.astype(np.float64)), 0)
            else:
                s = (np.abs(part).max(0) / 7).astype(np.float32)
                z = np.full(N, 8.0)
            bad = ~np.isfinite(part).all(0)
            s[bad] = np.nan
            z = np.where(bad, 0 if zero_points else 8, np.clip(z, 0, 15))
            steps = np.where(s > 0, np.rint(part / s.astype(np.float64)), 0)
            q[g * group:(g + 1) * group] = np.where(bad, z, np.clip(steps + z, 0, 15))
            scales[g], zeros[g] = s, z
    return q, scales, zeros


def _check_quantized(torch, W, group, zero_points):
    import clusternet_amd as cn
    K, N = W.shape
    w4 = cn.quantize_4bit(W, group=group, zero_points=zero_points)
    q, scales, zeros = _definition(W.double().cpu().numpy(), group, zero_points)
    got, padded = _codes(w4.codes, K, N)
    assert np.array_equal(w4.scales.cpu().numpy(), scales, equal_nan=True)
    if zero_points:
        assert np.array_equal(w4.zeros.cpu().numpy(), zeros)
    else:
        assert w4.zeros is None
    assert np.array_equal(got, q) and padded
    spread = lambda x: np.repeat(x, group, 0)[:K]  # noqa: E731
    back = (q - spread(zeros)).astype(np.float32) * spread(scales)
    assert np.array_equal(cn.dequantize_4bit(w4).cpu().numpy(), back, equal_nan=True)
    for dtype in (torch.float16, torch.bfloat16):
        assert torch.equal(cn.dequantize_4bit(w4, dtype=dtype).nan_to_num(7.0), torch.from_numpy(back).to(dtype).cuda().nan_to_num(7.0))
    return w4


@pytest.mark.parametrize("K,N", [(1, 1), (31, 15), (32, 16), (128, 64), (129, 65), (200, 17), (257, 100), (1000, 130)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zero_points", [False, True])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_quantisation_by_its_definition(torch, K, N, group, zero_points, dtype):
    rng = np.random.default_rng(K + N + group)
    W = torch.from_numpy(rng.normal(0.01, 0.05, (K, N)).astype(np.float32)).cuda().to(getattr(torch, dtype))
    _check_quantized(torch, W, group, zero_points)


@pytest.mark.parametrize("zero_points", [False, True])
def test_quantisation_at_its_borders(torch, zero_points):
    """Halves of a step (which go to the even code), groups of zeros, of one sign, of the smallest numbers and of very large ones,
    and groups with something that is not finite."""
    rng = np.random.default_rng(1)
    K, N = 256, 40
    w = rng.normal(0, 1, (K, N)).astype(np.float32)
    for c in range(12):  # steps of exactly 2^(c - 6): codes on and between borders
        w[:, c] = rng.integers(-14, 15, K) * 0.5 * 2.0 ** (c - 6)
        w[::32, c] = 7.0 * 2.0 ** (c - 6)
        if zero_points:
            w[1::32, c] = -8.0 * 2.0 ** (c - 6)
    for c in range(12, 16):  # just beside the borders
        w[:, c] = np.nextafter(((rng.integers(-7, 7, K) + 0.5) * 0.37).astype(np.float32), np.float32((-9.0, 9.0)[c % 2]))
        w[::32, c] = 7 * np.float32(0.37)
    w[:, 16] = 0.0
    w[:, 17] = -0.0
    w[:, 18] = np.abs(w[:, 18])
    w[:, 19] = -np.abs(w[:, 19])
    w[:, 20] *= 1e-44
    w[:, 21] *= 1e-38
    w[:, 22] *= 1e-30
    w[:, 23] = np.clip(w[:, 23], -3, 3) * np.float32(1e38)
    w[5, 24], w[200, 25], w[77, 26] = np.nan, np.inf, -np.inf
    w[:, 27] = 1e-45
    _check_quantized(torch, torch.from_numpy(w).cuda(), 32, zero_points)
    _check_quantized(torch, torch.from_numpy(w).cuda(), 128, zero_points)


def test_quantisation_of_a_part_of_a_matrix(torch):
    rng = np.random.default_rng(2)
    wide = torch.from_numpy(rng.normal(0, 1, (300, 90)).astype(np.float32)).cuda()
    import clusternet_amd as cn
    w4 = _check_quantized(torch, wide[7:207, 3:80], 64, True)
    back = torch.full((203, 85), 7.0, device="cuda")
    cn.dequantize_4bit(w4, out=back[1:201, 5:82])
    assert torch.equal(back[1:201, 5:82], cn.dequantize_4bit(w4))
    back[1:201, 5:82] = 7.0
    assert bool((back == 7.0).all())


@pytest.mark.parametrize("dtype,K,N", [("float32", 16500, 4100), ("bfloat16", 16500, 8200), ("float16", 8300, 16400)])
def test_weights_larger_than_the_caches(torch, dtype, K, N):
    """What the small sizes hold to the definition, at a size that is written past the caches: the same numbers as from 128
    rows at a time."""
    import clusternet_amd as cn
    gen = torch.Generator(device="cuda").manual_seed(K)
    W = (0.05 * torch.randn(K, N, device="cuda", generator=gen)).to(getattr(torch, dtype))
    for zero_points in (False, True):
        whole = cn.dequantize_4bit(cn.quantize_4bit(W, 64, zero_points), dtype=W.dtype)
        for first in (0, 128, K // 256 * 128, K // 128 * 128):
            part = W[first:first + 128].contiguous()
            assert torch.equal(whole[first:first + 128], cn.dequantize_4bit(cn.quantize_4bit(part, 64, zero_points), dtype=W.dtype))
        assert bool((whole.float() - W.float()).abs().max() <= 0.05)  # steps of a seventh of up to 0.35


def _weights(torch, rng, K, N, group, zero_points, whole):
    import clusternet_amd as cn
    groups = -(-K // group)
    q = rng.integers(0, 16, (K, N))
    scales = (2.0 ** rng.integers(-3, 3, (groups, N)) if whole else rng.uniform(0.001, 0.02, (groups, N))).astype(np.float32)
    zeros = rng.integers(0, 16, (groups, N)).astype(np.uint8) if zero_points else None
    w4 = cn.W4(torch.from_numpy(_stored(q)).cuda(), torch.from_numpy(scales).cuda(),
               None if zeros is None else torch.from_numpy(zeros).cuda(), K, N, group)
    spread = lambda x: np.repeat(x.astype(np.float64), group, 0)[:K]  # noqa: E731
    s = spread(scales)
    return w4, (q - (8 if zeros is None else spread(zeros))) * s, s


SIZES = [(1, 1, 1), (1, 128, 16), (1, 5, 33), (3, 127, 15), (16, 128, 64), (17, 130, 70), (13, 500, 199), (1, 4096, 1024), (33, 260, 48),
         (64, 1000, 130), (65, 384, 100), (200, 129, 17), (2, 1056, 16400), (5, 200, 33000), (20, 264, 16390),
         (40, 390, 8210), (300, 136, 1650)]


@pytest.mark.parametrize("M,K,N", SIZES)
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("group,zero_points", [(32, True), (64, False), (128, True), (128, False)])
def test_product(torch, M, K, N, dtype, group, zero_points):
    import clusternet_amd as cn
    rng = np.random.default_rng(M + K + N + group)
    # whole numbers: |a| <= 4, |q - z| s <= 60, sums below 2^24 / 8 for K <= 4096 / 2, exact in fp32 whatever the order
    w4, w, _ = _weights(torch, rng, K, N, group, zero_points, True)
    if K <= 2048:
        a = rng.integers(-4, 5, (M, K)).astype(np.float32)
        out = cn.gemm_w4(torch.from_numpy(a).cuda().to(getattr(torch, dtype)), w4)
        want = torch.from_numpy(a.astype(np.float64) @ w).float().to(getattr(torch, dtype))
        assert torch.equal(out.cpu(), want)
    w4, w, s = _weights(torch, rng, K, N, group, zero_points, False)
    a = torch.from_numpy(rng.normal(0, 1, (M, K)).astype(np.float32)).cuda().to(getattr(torch, dtype))
    out = cn.gemm_w4(a, w4)
    ad = a.double().cpu().numpy()
    want = ad @ w
    bound = (128 + K / group + 16) * 2.0 ** -23 * 62 * (np.abs(ad) @ s)
    if dtype != "float32":
        bound = bound * (1 + HALF[dtype]) + HALF[dtype] * np.abs(want) + 2.0 ** -25
    off = np.abs(out.double().cpu().numpy() - want)
    assert out.dtype == a.dtype and (off <= bound).all(), float((off - bound).max())
    assert torch.equal(out, cn.gemm_w4(a, w4))


def test_product_keeps_all_bits_of_fp32(torch):
    """Rows of A with a single number: the product has three exact parts of it and one rounded scale.  Numbers with all 24 bits
    set, tiny and huge ones."""
    import clusternet_amd as cn
    rng = np.random.default_rng(4)
    K = N = 64
    w4, w, s = _weights(torch, rng, K, N, 32, True, True)
    a = np.zeros((K, K), np.float32)
    values = np.concatenate([np.float32(2 - 2.0 ** -23) * 2.0 ** rng.integers(-60, 60, K // 2), rng.normal(0, 1, K // 2)]).astype(np.float32)
    a[np.arange(K), np.arange(K)] = values
    out = cn.gemm_w4(torch.from_numpy(a).cuda(), w4).double().cpu().numpy()
    # a (16 + q) and (16 + z) a are each rounded to 24 bits before their difference: two roundings of at most 31 |a| s
    assert (np.abs(out - values[:, None].astype(np.float64) * w) <= 3 * 2.0 ** -24 * 31 * np.abs(values[:, None].astype(np.float64)) * s).all()


def test_product_in_strided_places(torch):
    """Rows of A and out in wider matrices, aligned for 16-byte loads and not, and what surrounds the output stays."""
    import clusternet_amd as cn
    rng = np.random.default_rng(6)
    w4, w, _ = _weights(torch, rng, 300, 77, 64, False, True)
    for dtype in (torch.float32, torch.bfloat16):
        for off in (0, 1, 8):
            wide = torch.from_numpy(rng.integers(-4, 5, (20, 328)).astype(np.float32)).cuda().to(dtype)
            a = wide[2:15, off:off + 300]
            back = torch.full((15, 90), 7.0, device="cuda", dtype=dtype)
            cn.gemm_w4(a, w4, out=back[1:14, off + 1:off + 78])
            assert torch.equal(back[1:14, off + 1:off + 78].cpu(), torch.from_numpy(a.double().cpu().numpy() @ w).float().to(dtype))
            back[1:14, off + 1:off + 78] = 7.0
            assert bool((back == 7.0).all())


def test_product_of_nothing_and_of_not_finite(torch):
    import clusternet_amd as cn
    rng = np.random.default_rng(7)
    w4, w, _ = _weights(torch, rng, 200, 40, 64, True, True)
    assert cn.gemm_w4(torch.empty(0, 200, device="cuda"), w4).shape == (0, 40)
    none = cn.quantize_4bit(torch.empty(0, 40, device="cuda"))
    assert torch.equal(cn.gemm_w4(torch.empty(3, 0, device="cuda"), none), torch.zeros(3, 40, device="cuda"))
    assert cn.gemm_w4(torch.empty(3, 7, device="cuda"), cn.quantize_4bit(torch.empty(7, 0, device="cuda"))).shape == (3, 0)
    a = torch.ones(4, 200, device="cuda")
    a[1, 3] = float("nan")
    a[2, 199] = float("inf")
    out = cn.gemm_w4(a, w4)
    assert bool(out[1:3].isnan().all()) and torch.equal(out[[0, 3]].double().cpu(), torch.from_numpy(np.ones((2, 200)) @ w))
    # a scale that is not finite is its column's own
    w4.scales[1, 9] = float("nan")
    out = cn.gemm_w4(torch.ones(2, 200, device="cuda"), w4)
    assert bool(out[:, 9].isnan().all()) and bool(out[:, [c for c in range(40) if c != 9]].isfinite().all())


def test_in_graphs_and_on_other_streams(torch):
    import clusternet_amd as cn
    rng = np.random.default_rng(8)
    sets = []
    for M, K, N in ((1, 512, 300), (20, 1000, 64)):
        w4 = _weights(torch, rng, K, N, 64, True, False)[0]
        a = torch.from_numpy(rng.normal(0, 1, (M, K)).astype(np.float32)).cuda()
        cn.gemm_w4(a, w4)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = cn.gemm_w4(a, w4)
        sets.append((a, w4, graph, got))
    side = torch.cuda.Stream()
    for _ in range(4):
        for a, w4, graph, got in sets:
            a.mul_(-1.5)
            want = cn.gemm_w4(a, w4)
            with torch.cuda.stream(side):
                side.wait_stream(torch.cuda.default_stream())
                beside = cn.gemm_w4(a, w4)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want) and torch.equal(beside, want)
