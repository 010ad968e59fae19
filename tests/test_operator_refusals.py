"""Calls that the word-table, update and 4-bit operators refuse, checked without a GPU: the C entry points look at their
arguments before they need a device (the addresses here are never read), the binding before it calls them."""
import pytest

import clusternet_amd as cn

SHAPE, NULL, ARG, WORKSPACE, NO_DEVICE = 2, 1, 6, 5, 3
AT = 4096  # an address that no call gets as far as reading


def _refused(status, want):
    assert status == want, (status, cn.lib().cn_last_error())
    assert cn.lib().cn_last_error() != b""


def test_embedding_refuses():
    f = cn.lib().cn_embedding
    _refused(f(AT, 3, 4, 4, 4, AT, 32, 4, 1.0, AT, 4, None), ARG)        # no such type
    _refused(f(AT, 0, -1, 4, 4, AT, 32, 4, 1.0, AT, 4, None), SHAPE)
    _refused(f(AT, 0, 4, 4, 3, AT, 32, 4, 1.0, AT, 4, None), SHAPE)      # leading dimensions
    _refused(f(AT, 0, 4, 4, 4, AT, 32, 4, 1.0, AT, 3, None), SHAPE)
    _refused(f(AT, 0, 4, 4, 4, AT, 16, 4, 1.0, AT, 4, None), ARG)        # 16-bit tokens
    _refused(f(AT, 0, 4, 4, 4, AT, 32, -4, 1.0, AT, 4, None), SHAPE)
    _refused(f(AT, 0, 4, 4, 4, AT, 32, 2 ** 31, 1.0, AT, 4, None), SHAPE)
    _refused(f(AT, 0, 2 ** 31, 4, 4, AT, 32, 4, 1.0, AT, 4, None), SHAPE)
    _refused(f(None, 0, 4, 4, 4, AT, 32, 4, 1.0, AT, 4, None), NULL)
    _refused(f(AT, 0, 4, 4, 4, None, 32, 4, 1.0, AT, 4, None), NULL)
    _refused(f(AT, 0, 4, 4, 4, AT, 32, 4, 1.0, None, 4, None), NULL)
    assert f(None, 0, 0, 4, 4, None, 32, 0, 1.0, None, 4, None) == 0     # no tokens: nothing to do
    _refused(f(AT, 0, 4, 4, 4, AT, 32, 4, 1.0, AT, 4, None), ARG)        # into the table itself
    # more workgroups than a launch may have
    _refused(f(AT, 0, 4, 2048, 2048, AT, 32, 2 ** 27, 1.0, 2 * AT, 2048, None), SHAPE)
    _refused(f(AT, 0, 4, 2 ** 26 + 1, 2 ** 27, AT, 32, 4, 1.0, 2 * AT, 2 ** 27, None), SHAPE)


def test_embedding_grad_refuses():
    L = cn.lib()
    f, need = L.cn_embedding_grad, L.cn_embedding_grad_workspace_bytes
    size = need(3000, 50, 8)
    assert size > 3000 * 16 and need(0, 50, 8) == 0 and need(3000, 50, 0) == 0 and need(-1, 50, 8) == 0 and need(100, 50, 8) == 0
    ok = [AT, 0, 8, AT, 32, 3000, 50, 8, 1.0, 0, AT, 0, 8, AT, size, None]

    def call(**change):
        a = list(ok)
        for k, v in change.items():
            a[int(k[1:])] = v
        return f(*a)
    _refused(call(_1=7), ARG)
    _refused(call(_1=1, _11=2), ARG)          # fp16 errors, bf16 gradient
    _refused(call(_11=1), ARG)                # fp32 errors, fp16 gradient
    _refused(call(_2=7), SHAPE)
    _refused(call(_12=7), SHAPE)
    _refused(call(_4=8), ARG)
    _refused(call(_5=-1), SHAPE)
    _refused(call(_6=-1), SHAPE)
    _refused(call(_7=-1), SHAPE)
    _refused(call(_6=2 ** 31), SHAPE)
    for place in ("_0", "_3", "_10", "_13"):
        _refused(call(**{place: None}), NULL)
    _refused(call(_14=size - 1), WORKSPACE)
    _refused(call(_13=AT + 16), ARG)          # alignment of the workspace
    assert call(_5=0, _9=1, _0=None, _3=None, _13=None, _14=0) == 0
    _refused(call(), ARG)                     # onto the errors
    big = need(3000, 2 ** 30, 8)
    _refused(call(_10=2 * AT, _6=2 ** 30, _14=big), SHAPE)             # 2^25 workgroups that write zeros
    _refused(call(_10=2 * AT, _9=1, _7=2 ** 22 + 64, _2=2 ** 23, _12=2 ** 23, _14=2 ** 62), SHAPE)


def test_binding_refuses_tensors_of_the_host():
    torch = pytest.importorskip("torch")
    table, tokens = torch.zeros(4, 4), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(TypeError):
        cn.embedding(table, tokens)
    with pytest.raises(TypeError):
        cn.embedding_grad(table, tokens, 4)


def test_orthogonalize_refuses():
    L = cn.lib()
    need = L.cn_orthogonalize_workspace_bytes
    size = need(10, 20)
    assert size > 0 and need(20, 10) == size and need(0, 4) == 0 and need(4, 0) == 0 and need(-1, 4) == 0 and need(2 ** 17 + 1, 4) == 0
    ok = [AT, 0, 10, 20, 20, 5, AT, 0, 20, AT, size, None]

    def call(**change):
        a = list(ok)
        for k, v in change.items():
            a[int(k[1:])] = v
        return L.cn_orthogonalize(*a)
    _refused(call(_1=3), ARG)
    _refused(call(_7=-1), ARG)
    _refused(call(_2=-1), SHAPE)
    _refused(call(_3=-1), SHAPE)
    _refused(call(_2=2 ** 17 + 1), SHAPE)
    _refused(call(_4=19), SHAPE)
    _refused(call(_8=19), SHAPE)
    _refused(call(_5=0), ARG)
    _refused(call(_5=101), ARG)
    for place in ("_0", "_6", "_9"):
        _refused(call(**{place: None}), NULL)
    _refused(call(_10=size - 1), WORKSPACE)
    _refused(call(_9=AT + 128), ARG)
    assert call(_2=0, _0=None, _6=None, _9=None) == 0


def test_muon_update_refuses():
    L = cn.lib()
    size = L.cn_orthogonalize_workspace_bytes(10, 20)
    ok = [AT, 20, AT, 0, 20, AT, 20, 10, 20, 0.9, 1, 0.1, 0.0, 5, AT, size, None]

    def call(**change):
        a = list(ok)
        for k, v in change.items():
            a[int(k[1:])] = v
        return L.cn_muon_update(*a)
    _refused(call(_3=5), ARG)
    for place in ("_1", "_4", "_6"):
        _refused(call(**{place: 19}), SHAPE)
    _refused(call(_7=-1), SHAPE)
    _refused(call(_13=0), ARG)
    for place in ("_0", "_2", "_5", "_14"):
        _refused(call(**{place: None}), NULL)
    _refused(call(_15=size - 1), WORKSPACE)
    for places in ({}, {"_0": 2 * AT}, {"_2": 2 * AT}, {"_5": 2 * AT}):  # two or all of them the same matrix
        _refused(call(**places), ARG)
    assert call(_8=0, _0=None, _2=None, _5=None, _14=None) == 0


def test_w4_refuses():
    L = cn.lib()
    assert L.cn_w4_code_words(128, 16) == 256 and L.cn_w4_code_words(129, 17) == 4 * 256
    assert L.cn_w4_code_words(0, 16) == 0 and L.cn_w4_code_words(16, -1) == 0

    def caller(f, ok):
        def call(**change):
            a = list(ok)
            for k, v in change.items():
                a[int(k[1:])] = v
            return f(*a)
        return call
    q = caller(L.cn_quantize_4bit, [AT, 0, 64, 32, 32, 32, AT, AT, AT, None])
    _refused(q(_1=9), ARG)
    _refused(q(_2=-1), SHAPE)
    _refused(q(_3=-1), SHAPE)
    _refused(q(_4=31), SHAPE)
    for group in (0, -32, 16, 48, 256):
        _refused(q(_5=group), ARG)
    for place in ("_0", "_6", "_7"):
        _refused(q(**{place: None}), NULL)
    _refused(q(_6=AT + 4), ARG)
    _refused(q(_2=2 ** 31), SHAPE)
    assert q(_2=0, _0=None, _6=None, _7=None) == 0
    d = caller(L.cn_dequantize_4bit, [AT, AT, AT, 64, 32, 32, AT, 0, 32, None])
    _refused(d(_7=9), ARG)
    _refused(d(_5=33), ARG)
    _refused(d(_8=31), SHAPE)
    for place in ("_0", "_1", "_6"):
        _refused(d(**{place: None}), NULL)
    _refused(d(_0=AT + 8), ARG)
    g = caller(L.cn_gemm_w4, [4, 32, 64, AT, 0, 64, AT, AT, AT, 32, AT, 32, None])
    _refused(g(_4=9), ARG)
    _refused(g(_0=-1), SHAPE)
    _refused(g(_1=-1), SHAPE)
    _refused(g(_2=-1), SHAPE)
    _refused(g(_5=63), SHAPE)
    _refused(g(_11=31), SHAPE)
    _refused(g(_9=96), ARG)
    _refused(g(_0=2 ** 20 + 1), SHAPE)
    for place in ("_3", "_6", "_7", "_10"):
        _refused(g(**{place: None}), NULL)
    _refused(g(_6=AT + 8), ARG)
    _refused(g(), ARG)                        # the output is A
    _refused(g(_10=2 * AT, _1=2 ** 30, _11=2 ** 30), SHAPE)
    assert g(_0=0, _3=None, _6=None, _7=None, _10=None) == 0


def test_w4_binding_refuses():
    torch = pytest.importorskip("torch")
    with pytest.raises(TypeError):
        cn.quantize_4bit(torch.zeros(32, 16))
    with pytest.raises(TypeError):
        cn.W4(torch.zeros(1, 1, 64, 4, dtype=torch.int32), torch.zeros(1, 16), None, 32, 16, 32)
    with pytest.raises(TypeError):
        cn.orthogonalize(torch.zeros(3, 3))
    with pytest.raises(TypeError):
        cn.muon_update(torch.zeros(3, 3), torch.zeros(3, 3), torch.zeros(3, 3), 0.9, 0.1)
