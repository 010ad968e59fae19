"""The operators for models that read words, train with matrix updates and answer from 4-bit weights, as they are measured.

Each case is one call of an operator on synthetic data of the kind it meets: token numbers with the frequencies of text (the r-th
most frequent of V words appears with probability log(1 + 1/r) / log(V + 1)), gradients with a few strong directions in noise,
weights of the usual spread.  `run` computes a case in plain torch, or, where `own` is true, through clusternet_amd.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
NS_A, NS_B, NS_C = 3.4445, -4.7750, 2.0315
NS_STEPS = 5


def listed():
    return [
        # one batch of the reference's window language model: 128 windows of 11 words on its vocabulary
        {"name": "lookup 128 windows of 11", "op": "embedding", "rows": 100002, "cols": 120, "count": 1408, "dtype": "f32",
         "index": 64, "invalid": 0.0, "scale": 1.0},
        # a long training batch on a wide table, scaled by sqrt(cols), a few positions padded
        {"name": "lookup 65536 x 2048", "op": "embedding", "rows": 100002, "cols": 2048, "count": 65536, "dtype": "bf16",
         "index": 32, "invalid": 0.03, "scale": 45.25},
        # the same batches on the way back: the table updated in place, and the whole gradient for an optimiser
        {"name": "grad 128 windows of 11, added", "op": "embedding_grad", "rows": 100002, "cols": 120, "count": 1408,
         "dtype": "f32", "index": 64, "invalid": 0.0, "scale": -0.1, "accumulate": True},
        {"name": "grad 65536 x 2048, whole", "op": "embedding_grad", "rows": 100002, "cols": 2048, "count": 65536,
         "dtype": "bf16", "index": 32, "invalid": 0.03, "scale": 45.25, "accumulate": False},
        # the update of a small first layer, and of a wide one kept in 16 bits
        {"name": "orthogonalize 784 x 1024", "op": "orthogonalize", "rows": 784, "cols": 1024, "dtype": "f32"},
        {"name": "orthogonalize 4096 x 16384", "op": "orthogonalize", "rows": 4096, "cols": 16384, "dtype": "bf16"},
        # a whole weight update: an odd layer, and a square one of the 8-bit benchmark's size
        {"name": "muon 4001 x 1000", "op": "muon", "rows": 4001, "cols": 1000, "dtype": "f32"},
        {"name": "muon 4096 x 4096", "op": "muon", "rows": 4096, "cols": 4096, "dtype": "bf16"},
        # trained weights to 4 bits and back: a layer with zero points, and a large one
        {"name": "4-bit round trip 4096 x 4096", "op": "round_trip", "inner": 4096, "outer": 4096, "group": 64,
         "zero_points": True, "dtype": "f32"},
        {"name": "4-bit round trip 16384 x 8192", "op": "round_trip", "inner": 16384, "outer": 8192, "group": 128,
         "zero_points": False, "dtype": "bf16"},
        # answers: a handful of rows through an odd layer, and one token through a large one
        {"name": "gemm_w4 13 x 5000 x 1999", "op": "gemm_w4", "count": 13, "inner": 5000, "outer": 1999, "group": 64,
         "zero_points": True, "dtype": "f32"},
        {"name": "gemm_w4 1 x 16384 x 16384", "op": "gemm_w4", "count": 1, "inner": 16384, "outer": 16384, "group": 128,
         "zero_points": False, "dtype": "bf16"},
    ]


def draw(rng):
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(("embedding", "embedding_grad", "orthogonalize", "muon", "round_trip", "gemm_w4"))
    dtype = rng.choice(("f32", "f16", "bf16"))
    if op in ("embedding", "embedding_grad"):
        case = {"op": op, "rows": size(1000, 100002), "cols": size(16, 2048), "count": size(1, 65536), "dtype": dtype,
                "index": rng.choice((32, 64)), "invalid": rng.choice((0.0, 0.05)), "scale": round(rng.uniform(0.5, 40.0), 3)}
        if op == "embedding_grad":
            case["accumulate"] = rng.random() < 0.5
        return case
    if op in ("orthogonalize", "muon"):
        rows, cols = size(16, 4096), size(16, 16384 if op == "orthogonalize" else 4096)
        if rng.random() < 0.5:
            rows, cols = cols, rows
        return {"op": op, "rows": rows, "cols": cols, "dtype": "f32" if dtype == "f16" else dtype}
    inner, outer = size(128, 8192), size(64, 16384)
    case = {"op": op, "inner": inner, "outer": outer, "group": rng.choice((32, 64, 128)), "zero_points": rng.random() < 0.5,
            "dtype": dtype}
    if op == "gemm_w4":
        case["count"] = size(1, 64)
    return case


# ---- inputs -------------------------------------------------------------------------------------------------------
def _tokens(case, gen):
    """Token numbers with the frequencies of text, most frequent first; a share of positions names no row (-1)."""
    u = torch.rand(case["count"], generator=gen, device="cuda", dtype=torch.float64)
    tokens = ((u * math.log(case["rows"] + 1)).exp().floor().long() - 1).clamp_(0, case["rows"] - 1)
    if case["invalid"]:
        tokens[torch.rand(case["count"], generator=gen, device="cuda") < case["invalid"]] = -1
    return tokens.to(torch.int32 if case["index"] == 32 else torch.int64)


def _gradient(rows, cols, gen):
    """Eight strong directions in noise."""
    strong = torch.randn(rows, 8, generator=gen, device="cuda") @ torch.randn(8, cols, generator=gen, device="cuda")
    return (0.02 * strong + 0.05 * torch.randn(rows, cols, generator=gen, device="cuda")) * 1e-2


def _columns(case):
    """Columns and rows of the stored form: whole tiles of 16 columns and 128 rows."""
    return -(-case["outer"] // 16), -(-case["inner"] // 128)


def _pack(q):
    """The stored form of 4-bit codes q (K x N): int32 words [N / 16][K / 128][64][4], nibble i of word t of lane l is row
    128 b + 32 t + 8 (l / 16) + i, column 16 a + l % 16; rows and columns past the matrix hold 0."""
    K, N = q.shape
    nt, kb = -(-N // 16), -(-K // 128)
    full = torch.zeros(kb * 128, nt * 16, dtype=torch.int64, device=q.device)
    full[:K, :N] = q
    v = full.view(kb, 4, 4, 8, nt, 16).permute(4, 0, 2, 5, 1, 3)  # a, b, h, column, t, i
    words = (v << (4 * torch.arange(8, device=q.device))).sum(-1)
    words = torch.where(words >= 2 ** 31, words - 2 ** 32, words)
    return words.to(torch.int32).reshape(nt, kb, 64, 4).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    op, s = case["op"], dict(case)
    dt = DTYPES[case["dtype"]]
    if op == "embedding":
        s["table"] = torch.empty(case["rows"], case["cols"], device="cuda", dtype=dt).normal_(0, 0.02, generator=gen)
        s["tokens"] = _tokens(case, gen)
    elif op == "embedding_grad":
        s["error"] = torch.empty(case["count"], case["cols"], device="cuda", dtype=dt).normal_(0, 0.01, generator=gen)
        s["tokens"] = _tokens(case, gen)
        if case["accumulate"]:
            s["table"] = torch.empty(case["rows"], case["cols"], device="cuda").normal_(0, 0.02, generator=gen)
    elif op == "orthogonalize":
        s["grad"] = _gradient(case["rows"], case["cols"], gen).to(dt)
    elif op == "muon":
        s["grad"] = _gradient(case["rows"], case["cols"], gen).to(dt)
        s["momentum"] = 5 * _gradient(case["rows"], case["cols"], gen)
        bound = math.sqrt(6.0 / (case["rows"] + case["cols"]))
        s["w"] = torch.empty(case["rows"], case["cols"], device="cuda").uniform_(-bound, bound, generator=gen)
    elif op == "round_trip":
        s["w"] = torch.empty(case["inner"], case["outer"], device="cuda", dtype=dt).normal_(0, 0.02, generator=gen)
    else:
        K, N, g = case["inner"], case["outer"], case["group"]
        groups = -(-K // g)
        q = torch.randn(K, N, generator=gen, device="cuda").mul_(3).add_(8).round_().clamp_(0, 15)
        s["codes"] = _pack(q)
        s["scales"] = torch.empty(groups, N, device="cuda").uniform_(0.002, 0.008, generator=gen)
        s["zeros"] = torch.randint(6, 11, (groups, N), generator=gen, device="cuda", dtype=torch.uint8) if case["zero_points"] else None
        s["x"] = torch.empty(case["count"], K, device="cuda", dtype=dt).normal_(0, 1, generator=gen)
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------
def _plain_newton_schulz(u):
    x = u.t() if u.shape[0] > u.shape[1] else u
    x = x / (x.double().norm().float() + 1e-7)
    for _ in range(NS_STEPS):
        a = x @ x.t()
        x = NS_A * x + (NS_B * a + NS_C * (a @ a)) @ x
    return x.t() if u.shape[0] > u.shape[1] else x


def _unpack(codes, K, N):
    nt, kb = codes.shape[:2]
    nibbles = (codes.view(nt, kb, 4, 16, 4, 1) >> (4 * torch.arange(8, device=codes.device, dtype=torch.int32))) & 15
    return nibbles.permute(1, 4, 2, 5, 0, 3).reshape(kb * 128, nt * 16)[:K, :N]


def _spread(v, g, K):
    """One value per group of g rows, for each of the K rows."""
    return v.repeat_interleave(g, 0)[:K]


def _plain(s):
    op = s["op"]
    if op == "embedding":
        t = s["tokens"].long()
        named = (t >= 0) & (t < s["rows"])
        y = s["table"][t.clamp(0, s["rows"] - 1)].float() * s["scale"]
        return torch.where(named[:, None], y, torch.zeros((), device="cuda")).to(s["table"].dtype)
    if op == "embedding_grad":
        t = s["tokens"].long()
        named = (t >= 0) & (t < s["rows"])
        e = torch.where(named[:, None], s["error"].float(), torch.zeros((), device="cuda")) * s["scale"]
        out = s["table"] if s["accumulate"] else torch.zeros(s["rows"], s["cols"], device="cuda")
        return out.index_add_(0, t.clamp(0, s["rows"] - 1), e)
    if op == "orthogonalize":
        return _plain_newton_schulz(s["grad"].float()).to(s["grad"].dtype)
    if op == "muon":
        g = s["grad"].float()
        s["momentum"].mul_(0.95).add_(g)
        o = _plain_newton_schulz(g + 0.95 * s["momentum"])
        s["w"].mul_(1 - 0.05 * 0.01).sub_(0.05 * o)
        return [s["w"], s["momentum"]]
    if op == "round_trip":
        K, N, g = s["inner"], s["outer"], s["group"]
        groups = -(-K // g)
        w = torch.full((groups * g, N), float("nan"), device="cuda")
        w[:K] = s["w"]
        w = w.view(groups, g, N)
        # a code next to a border is decided in 64 bits
        if s["zero_points"]:
            top = torch.where(w.isnan(), torch.zeros_like(w), w).amax(1)
            low = torch.where(w.isnan(), torch.zeros_like(w), w).amin(1)
            scale = ((top.double() - low.double()) / 15).float()
            zero = (-low.double() / scale.double()).round().clamp(0, 15)
        else:
            scale = (torch.where(w.isnan(), torch.zeros_like(w), w).abs().amax(1).double() / 7).float()
            zero = torch.full((groups, N), 8.0, device="cuda", dtype=torch.float64)
        q = ((w.double() / scale.double()[:, None]).round() + zero[:, None]).clamp(0, 15) - zero[:, None]
        back = (q.float() * scale[:, None]).reshape(groups * g, N)[:K]
        return [back, scale] + ([zero.to(torch.uint8)] if s["zero_points"] else [])
    K, N, g = s["inner"], s["outer"], s["group"]
    zero = 8.0 if s["zeros"] is None else _spread(s["zeros"].float(), g, K)
    w = (_unpack(s["codes"], K, N).float() - zero) * _spread(s["scales"], g, K)
    return (s["x"].float() @ w).to(s["x"].dtype)


def _own(s):
    import clusternet_amd as cn
    op = s["op"]
    if op == "embedding":
        return cn.embedding(s["table"], s["tokens"], scale=s["scale"])
    if op == "embedding_grad":
        if s["accumulate"]:
            return cn.embedding_grad(s["error"], s["tokens"], s["rows"], scale=s["scale"], out=s["table"], accumulate=True)
        return cn.embedding_grad(s["error"], s["tokens"], s["rows"], scale=s["scale"], out_dtype=torch.float32)
    if op == "orthogonalize":
        return cn.orthogonalize(s["grad"])
    if op == "muon":
        cn.muon_update(s["momentum"], s["grad"], s["w"], 0.95, 0.05, nesterov=True, weight_decay=0.01)
        return [s["w"], s["momentum"]]
    if op == "round_trip":
        w4 = cn.quantize_4bit(s["w"], group=s["group"], zero_points=s["zero_points"])
        back = cn.dequantize_4bit(w4)
        return [back, w4.scales] + ([w4.zeros] if s["zero_points"] else [])
    w4 = cn.W4(s["codes"], s["scales"], s["zeros"], s["inner"], s["outer"], s["group"])
    return cn.gemm_w4(s["x"], w4)


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def _distinct(case):
    """Expected number of distinct rows that the tokens of a case name."""
    r = np.arange(1, case["rows"] + 1, dtype=np.float64)
    p = np.log1p(1 / r) / math.log(case["rows"] + 1) * (1 - case["invalid"])
    return float(-np.expm1(case["count"] * np.log1p(-p)).sum())


def work(case):
    op = case["op"]
    es = BYTES[case["dtype"]]
    if op == "embedding":
        return {"bytes": _distinct(case) * case["cols"] * es + case["count"] * (case["cols"] * es + case["index"] // 8), "flops": 0}
    if op == "embedding_grad":
        into = 2 * _distinct(case) if case["accumulate"] else case["rows"]
        return {"bytes": case["count"] * (case["cols"] * es * (1 - case["invalid"]) + case["index"] // 8) + into * case["cols"] * 4,
                "flops": case["count"] * case["cols"]}
    if op in ("orthogonalize", "muon"):
        m, n = sorted((case["rows"], case["cols"]))
        flops = NS_STEPS * (3.0 * m * m * n + 1.0 * m * m * m)  # the symmetric products by their half
        return {"bytes": m * n * (2 * es if op == "orthogonalize" else es + 16), "flops": flops}
    K, N, g = case["inner"], case["outer"], case["group"]
    side = -(-K // g) * N * (5 if case["zero_points"] else 4)
    if op == "round_trip":
        return {"bytes": K * N * (es + 4) + side, "flops": 0}
    return {"bytes": K * N / 2 + side + case["count"] * (K + N) * es, "flops": 2.0 * case["count"] * K * N}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------
def _exact_orthogonal(u):
    flip = u.shape[0] > u.shape[1]
    x = u.T.contiguous() if flip else u
    x = x / (torch.sqrt((x * x).sum()) + 1e-7)
    for _ in range(NS_STEPS):
        xt = x.T.contiguous()
        gram = torch.matmul(x, xt)
        x = NS_A * x + NS_B * torch.matmul(gram, x) + NS_C * torch.matmul(gram, torch.matmul(gram, x))
    return x.T if flip else x


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("embedding", "embedding_grad"):
        t = s["tokens"].to(torch.int64)
        at = torch.nonzero((t >= 0) & (t < case["rows"])).flatten()
        if op == "embedding":
            out = torch.zeros(case["count"], case["cols"], dtype=torch.float64, device="cuda")
            out[at] = s["table"].index_select(0, t[at]).double() * case["scale"]
            return out
        out = s["table"].double() if case["accumulate"] else torch.zeros(case["rows"], case["cols"], dtype=torch.float64, device="cuda")
        return out.index_add_(0, t[at], s["error"].index_select(0, at).double() * case["scale"])
    if op == "orthogonalize":
        return _exact_orthogonal(s["grad"].double())
    if op == "muon":
        g = s["grad"].double()
        momentum = 0.95 * s["momentum"].double() + g
        return [(1 - 0.05 * 0.01) * s["w"].double() - 0.05 * _exact_orthogonal(g + 0.95 * momentum), momentum]
    K, N, g = case["inner"], case["outer"], case["group"]
    group_of_row = torch.arange(K, device="cuda") // g
    if op == "round_trip":
        w = s["w"].double()
        groups = -(-K // g)
        index = group_of_row[:, None].expand(K, N)
        zeros = torch.zeros(groups, N, dtype=torch.float64, device="cuda")
        if case["zero_points"]:
            high = zeros.scatter_reduce(0, index, w, "amax")
            low = zeros.scatter_reduce(0, index, w, "amin")
            scale = ((high - low) / 15).float().double()  # the stored scale is a number of 32 bits
            zero = torch.round(-low / scale).clamp(0, 15)
        else:
            scale = (zeros.scatter_reduce(0, index, w.abs(), "amax") / 7).float().double()
            zero = zeros + 8
        z = zero[group_of_row]
        q = (torch.round(w / scale[group_of_row]) + z).clamp(0, 15)
        return [(q - z) * scale[group_of_row], scale] + ([None] if case["zero_points"] else [])
    shifts = torch.arange(0, 32, 4, device="cuda")
    nt, kb = s["codes"].shape[0], s["codes"].shape[1]
    q = torch.bitwise_and(torch.bitwise_right_shift(s["codes"].long()[..., None], shifts), 15)  # [nt][kb][lane][t][i]
    q = q.reshape(nt, kb, 4, 16, 4, 8).permute(0, 3, 1, 4, 2, 5).reshape(nt * 16, kb * 128)[:N, :K].double()
    z = 8.0 if s["zeros"] is None else s["zeros"].double()[group_of_row].T
    w = (q - z) * s["scales"].double()[group_of_row].T
    return torch.matmul(s["x"].double(), w.T.contiguous())
