"""A decoder layer on the cache as a program runs it: projection of q, k and v
in one product, K and V written from its rows, attention over the cache,
output projection plus residual, and the MLP with its activation and residual;
a prompt first, then single tokens.  Each stage is held to 64 bits on the
inputs that the engine gave it."""
import numpy as np
import pytest

import kv_ref as ref
import oracle_lib as orc
import s3e
from test_gpu_mul_mat_act import U, activation, product64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t,wt", [(ref.Q4_0, orc.Q4_0), (ref.Q8_0, orc.F16)])
def test_prompt_then_tokens(ctx, t, wt):
    E, nh, heads, D, F, page = 256, 4, 2, 64, 512, 32
    rng = np.random.default_rng(17)
    qkv_n = (nh + 2 * heads) * D
    shapes = {"qkv": (qkv_n, E), "out": (E, nh * D), "fc1": (F, E), "fc2": (E, F)}
    wb = {k: orc.to_weight_bytes(wt, (rng.standard_normal(s) * 0.06).astype(np.float32)) for k, s in shapes.items()}
    w = {k: ctx.weight(wt, s[1], s[0], wb[k]) for k, s in shapes.items()}
    bias = {k: (0.1 * rng.standard_normal(s[0])).astype(np.float32) for k, s in shapes.items()}
    bd = {k: ctx.to_device(b) for k, b in bias.items()}
    prompts, steps = [45, 7], 3
    most = max(prompts) + steps
    ld = -(-most // page)
    n_pages = 2 * ld + 1
    c = s3e.KVCache(t, heads, D, page, n_pages)
    c = s3e.KVCache(t, heads, D, page, n_pages, ctx.to_device(rng.integers(0, 256, s3e.kv_cache_bytes(c), dtype=np.uint8)))
    table = rng.permutation(n_pages)[:2 * ld].reshape(2, ld).astype(np.int32)
    td = ctx.to_device(table)
    held = [[], []]  # K and V rows that went into each sequence
    lens = [0, 0]

    def product(name, x, M, act, residual=None):
        n = shapes[name][0]
        y = ctx.buffer(M * n * 4)
        ws = ctx.buffer(max(16, s3e.mul_mat_act_workspace(w[name], M)))
        ctx.mul_mat_act(w[name], x, M, y, ws, bias=bd[name], act=act, residual=residual)
        ctx.sync()
        X, Y = x.download(np.float32, (M, shapes[name][1])), y.download(np.float32, (M, n))
        p, mag = product64(wt, wb[name], n, shapes[name][1], X)
        p, mag = p + bias[name], mag + np.abs(bias[name])
        want = activation(act, p)
        bound = 1.13 * (shapes[name][1] + 16) * U * mag + 1e-6 * np.abs(p)
        if residual:
            R = residual.download(np.float32, (M, n))
            want, bound = want + R, bound + U * np.abs(want + R)
        assert (np.abs(Y - want) <= bound).all(), name
        return y, Y

    for step in range(1 + steps):
        nq = prompts if step == 0 else [1, 1]
        M = sum(nq)
        x = ctx.to_device(rng.standard_normal((M, E)).astype(np.float32))
        qkv, rows = product("qkv", x, M, "none")
        slots, row = [], 0
        for s, n in enumerate(nq):
            for i in range(n):
                j = lens[s] + i
                slots.append(table[s, j // page] * page + j % page)
                held[s].append(rows[row, nh * D:].reshape(2, heads, D))
                row += 1
            lens[s] += n
        sd = ctx.to_device(np.array(slots, np.int32))
        k, v = (s3e.DeviceView(qkv.ptr + 4 * (nh + i * heads) * D, 0) for i in range(2))
        starts = np.cumsum([0] + nq).astype(np.int32)
        ad = [ctx.to_device(starts), ctx.to_device(np.array(lens, np.int32))]
        b = s3e.KVBatch(2, M, max(nq), max(lens), *ad, td, ld)
        need = s3e.kv_attn_workspace(c, b, nh, s3e.TYPE_F32)
        ws, o = ctx.buffer(max(need, 16)), ctx.buffer(M * nh * D * 4)
        ctx.kv_write(c, s3e.TYPE_F32, k, (qkv_n, D), v, (qkv_n, D), sd, M)
        ctx.kv_attn(c, b, s3e.TYPE_F32, qkv, (qkv_n, D), nh, D ** -0.5, o, ws, causal=True)
        ctx.sync()
        got = o.download(np.float32, (M, nh, D))
        for s, n in enumerate(nq):
            kv = np.stack(held[s])
            parts = [p for i in range(2) for p in ref.quantize(t, kv[:, i])]
            see = np.arange(lens[s]) <= lens[s] - n + np.arange(n)[:, None]
            q = rows[starts[s]:starts[s + 1], :nh * D].reshape(n, nh, D)
            want, mag, A = ref.attention(t, *parts, q, D ** -0.5, see)
            bound = ref.attention_bound(True, want, mag, A, lens[s], D, ref.largest(t, *parts[2:]))
            off = np.abs(got[starts[s]:starts[s + 1]] - want)
            assert (off <= bound).all(), (step, s, (off / bound).max(), np.argwhere(off > bound)[:5])
        y, _ = product("out", o, M, "none", x)
        z, _ = product("fc1", y, M, "gelu_erf")
        product("fc2", z, M, "none", y)
