"""s3e_mul_mat_act: products with bias, activation and residual in their
epilogue, against 64 bits.

Bound of a value (u = 2^-24): the product's operands are the same integers and
fp16 (or fp32) values on both sides, so the sum differs by at most (K + 16)·u
of Σ|x·w| (a rounding a term, whatever the order; the bias among them); no
activation's slope exceeds 1.13; an activation's own evaluation is within
1e-6 of its argument (erfc to 3.1e-7 relative, exponential, reciprocal and
three products to u each); the residual's sum rounds once more.
"""
import ctypes

import numpy as np
import pytest
from scipy.special import erf

import kv_ref
import oracle_lib as orc
import s3e
from test_zz_no_alloc import _Graphs

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ALL = {"q4_0": orc.Q4_0, "q4_1": orc.Q4_1, "q8_0": orc.Q8_0, "f16": orc.F16, "f32": orc.F32}


def activation(name, y):
    if name == "relu":
        return np.maximum(y, 0)
    if name == "gelu_erf":
        return 0.5 * y * (1 + erf(y * np.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * y * (1 + np.tanh(np.sqrt(2 / np.pi) * (y + 0.044715 * y ** 3)))
    if name == "silu":
        return y / (1 + np.exp(-y))
    return y


def product64(t, wb, N, K, X):
    """W X in 64 bits from the weight's bytes and ggml's conversion of X, and Σ|x·w|."""
    if t in (orc.F32, orc.F16):
        W = np.asarray(wb).view(np.float32 if t == orc.F32 else np.float16).reshape(N, K).astype(np.float64)
        x = (X if t == orc.F32 else X.astype(np.float16)).astype(np.float64)
        return x @ W.T, np.abs(x) @ np.abs(W).T
    size = {orc.Q4_0: 18, orc.Q4_1: 20, orc.Q8_0: 34}[t]
    b = np.asarray(wb).view(np.uint8).reshape(N, K // 32, size)
    d = np.ascontiguousarray(b[..., :2]).view(np.float16)[..., 0].astype(np.float64)
    q, xd = kv_ref.quantize(kv_ref.Q8_0, X)
    x = kv_ref.values(kv_ref.Q8_0, q, xd)
    if t == orc.Q8_0:
        c = b[..., 2:].view(np.int8).astype(np.float64)
    else:
        n = b[..., size - 16:]
        c = np.concatenate([n & 15, n >> 4], -1).astype(np.float64) - (8 if t == orc.Q4_0 else 0)
    W = (c * d[..., None]).reshape(N, K)
    y, mag = x @ W.T, np.abs(x) @ np.abs(W).T
    if t == orc.Q4_1:
        m = np.ascontiguousarray(b[..., 2:4]).view(np.float16)[..., 0].astype(np.float64)
        top = np.abs(X.reshape(len(X), -1, 32)).max(-1)
        s = ((top / np.float32(127)) * q.reshape(len(X), -1, 32).astype(np.float32).sum(-1)).astype(np.float16).astype(np.float64)
        y, mag = y + s @ m.T, mag + np.abs(s) @ np.abs(m).T
    return y, mag


class Case:
    def __init__(self, ctx, t, M, N, K, bias, residual, seed):
        rng = np.random.default_rng(seed)
        self.M, self.N, self.K, self.t = M, N, K, t
        self.W = (rng.standard_normal((N, K)) * 0.05).astype(np.float32)
        self.X = rng.standard_normal((M, K)).astype(np.float32)
        self.wb = orc.to_weight_bytes(t, self.W)
        self.w = ctx.weight(t, K, N, self.wb)
        self.bias = rng.standard_normal(N).astype(np.float32) if bias else None
        self.R = rng.standard_normal((M, N)).astype(np.float32) if residual else None
        self.Xd = ctx.to_device(self.X)
        self.bd = ctx.to_device(self.bias) if bias else None
        self.Rd = ctx.to_device(self.R) if residual else None
        self.Y = ctx.to_device(np.full((M + 1, N), 7, np.float32))
        self.ws = ctx.to_device(np.full(s3e.mul_mat_act_workspace(self.w, M) + 16, 0xFF, np.uint8))  # NaN in every format

    def run(self, ctx, act, Y=None):
        ctx.mul_mat_act(self.w, self.Xd, self.M, Y or self.Y, self.ws, bias=self.bd, act=act, residual=self.Rd)

    def got(self, Y=None):
        return (Y or self.Y).download(np.float32, (self.M, self.N))

    def check(self, act, got):
        y, mag = product64(self.t, self.wb, self.N, self.K, self.X)
        if self.bias is not None:
            y, mag = y + self.bias, mag + np.abs(self.bias)
        want = activation(act, y)
        bound = 1.13 * (self.K + 16) * U * mag + 1e-6 * np.abs(y)
        if self.R is not None:
            want = want + self.R
            bound = bound + U * np.abs(want)
        off = np.abs(got - want)
        assert (off <= bound).all(), (off / bound).max()


SHAPES = [(1, 33, 32), (1, 1024, 4736), (7, 130, 224), (33, 64, 160), (64, 512, 1024), (65, 257, 96), (130, 1024, 1024),
          (300, 96, 1056), (1601, 256, 128)]


@pytest.mark.parametrize("name", ALL)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product_with_epilogue(ctx, name, M, N, K):
    for k, (act, bias, residual) in enumerate([("gelu_erf", True, False), ("none", True, True), ("silu", False, True),
                                               ("relu", True, True), ("gelu_tanh", True, False)]):
        if k != (M + N + len(name)) % 5 and k > 1:
            continue
        print(name, M, N, K, act, bias, residual, flush=True)
        c = Case(ctx, ALL[name], M, N, K, bias, residual, 7 * M + k)
        c.run(ctx, act)
        ctx.sync()
        c.check(act, c.got())
        assert (c.Y.download(np.float32, (M + 1, N))[M] == 7).all()
        c.w.free()


def test_wide_f16_product(ctx):
    # 128 x 128 tiles
    c = Case(ctx, orc.F16, 1300, 5120, 512, True, True, 3)
    c.run(ctx, "silu")
    ctx.sync()
    c.check("silu", c.got())


@pytest.mark.parametrize("name", ALL)
@pytest.mark.parametrize("M,N,K", [(5, 130, 256), (64, 96, 4736), (300, 512, 1024)])
def test_without_an_epilogue_it_is_mul_mat(ctx, name, M, N, K):
    c = Case(ctx, ALL[name], M, N, K, True, False, 5)
    c.run(ctx, "none")
    other = ctx.buffer(M * N * 4)
    ctx.mul_mat(c.w, c.Xd, M, other, c.bd)
    ctx.sync()
    assert np.array_equal(c.got(), c.got(other))


@pytest.mark.parametrize("name", ALL)
@pytest.mark.parametrize("M,N,K", [(5, 130, 256), (64, 96, 4736), (300, 512, 1024), (70, 130, 64)])
def test_residual_in_place(ctx, name, M, N, K):
    c = Case(ctx, ALL[name], M, N, K, True, True, 6)
    c.run(ctx, "silu")
    ctx.sync()
    want = c.got()
    c.run(ctx, "silu", c.Rd)
    ctx.sync()
    assert np.array_equal(c.got(c.Rd), want)


@pytest.mark.parametrize("act", [a for a in s3e.ACTS if a != "none"])
def test_activations_of_unusual_values(ctx, act):
    # a product with the identity: the activation of given values, far out and at the ends of fp32
    v = np.concatenate([np.linspace(-30, 30, 4001), [0.0, -0.0, 1e-30, -1e-30, 1e4, -1e4, 1e19, -1e19, 3e38, -3e38]]).astype(np.float32)
    K = 32
    X = np.zeros((len(v), K), np.float32)
    X[:, 0] = v
    W = np.eye(K, dtype=np.float32)
    w = ctx.weight(orc.F32, K, K, orc.to_weight_bytes(orc.F32, W))
    Xd, Y = ctx.to_device(X), ctx.buffer(len(v) * K * 4)
    ws = ctx.buffer(max(16, s3e.mul_mat_act_workspace(w, len(v))))
    ctx.mul_mat_act(w, Xd, len(v), Y, ws, act=act)
    ctx.sync()
    got = Y.download(np.float32, X.shape)[:, 0].astype(np.float64)
    with np.errstate(over="ignore"):
        want = activation(act, v.astype(np.float64))
    assert (np.abs(got - want) <= 1e-6 * np.abs(v)).all()


@pytest.mark.parametrize("name", ALL)
@pytest.mark.parametrize("M,N,K", [(7, 256, 2048), (300, 512, 1024)])
def test_captured_beside_another_graph(ctx, name, M, N, K):
    """Two captured products with workspaces of their own, replayed on two streams at once, beside eager products."""
    gr = _Graphs()
    gr.h.hipStreamCreateWithFlags.argtypes = [ctypes.POINTER(ctypes.c_void_p), ctypes.c_uint]
    gr.h.hipStreamSynchronize.argtypes = gr.h.hipStreamDestroy.argtypes = [ctypes.c_void_p]
    other = ctypes.c_void_p()
    assert gr.h.hipStreamCreateWithFlags(ctypes.byref(other), 1) == 0
    cases = [Case(ctx, ALL[name], M, N, K, True, True, 40 + i) for i in range(3)]
    want = []
    for c in cases:
        c.run(ctx, "gelu_tanh")
        ctx.sync()
        want.append(c.got())
        c.check("gelu_tanh", want[-1])
    graphs = [gr.capture(ctx.stream, lambda c=c: c.run(ctx, "gelu_tanh")) for c in cases[:2]]
    try:
        for rep in range(4):
            for c in cases:
                c.Y.upload(np.full((M, N), np.nan, np.float32))
            assert gr.h.hipGraphLaunch(graphs[0][1], ctx.stream) == 0
            assert gr.h.hipGraphLaunch(graphs[1][1], other) == 0
            cases[2].run(ctx, "gelu_tanh")
            ctx.sync()
            assert gr.h.hipStreamSynchronize(other) == 0
            for c, y in zip(cases, want):
                assert np.array_equal(c.got(), y), rep
    finally:
        for g, ex in graphs:
            gr.h.hipGraphExecDestroy(ex)
            gr.h.hipGraphDestroy(g)
        gr.h.hipStreamDestroy(other)


def test_refusals(ctx):
    c = Case(ctx, orc.Q4_0, 70, 64, 4096, True, True, 1)
    need = s3e.mul_mat_act_workspace(c.w, c.M)
    assert need > 0 and s3e.mul_mat_act_workspace(c.w, 0) == 0

    def call(**over):
        a = dict(ctx=ctx.handle, w=c.w.handle, X=c.Xd.ptr, M=c.M, bias=c.bd.ptr, act=2, R=c.Rd.ptr, Y=c.Y.ptr, ws=c.ws.ptr, n=need)
        a.update(over)
        return s3e.LIB.s3e_mul_mat_act(*a.values())

    INVALID, UNSUPPORTED = 1, 4
    for over in (dict(ctx=None), dict(w=None), dict(X=None), dict(Y=None), dict(M=-1), dict(act=-1), dict(act=5), dict(n=need - 1),
                 dict(ws=None), dict(ws=c.ws.ptr + 4), dict(X=c.Xd.ptr + 2), dict(Y=c.Xd.ptr), dict(Y=c.bd.ptr),
                 dict(R=c.Y.ptr + 4), dict(ws=c.Xd.ptr), dict(ws=c.Y.ptr)):
        assert call(**over) == INVALID, over
        assert s3e.LIB.s3e_last_error()
    for M in (262141, 1 << 40):
        assert call(M=M) == UNSUPPORTED
        with pytest.raises(s3e.S3EError):
            s3e.mul_mat_act_workspace(c.w, M)
    assert call(M=0) == 0 and call() == 0
    ctx.sync()
    odd = ctx.weight(orc.F32, 36, 64, np.zeros((64, 36), np.float32))  # K not whole blocks
    assert call(w=odd.handle) == UNSUPPORTED
