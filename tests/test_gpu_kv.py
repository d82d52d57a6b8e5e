"""The quantized key/value cache on the GPU: rows as they are written (every
byte, against the documented layout), rows read back, and attention over them
against 64-bit attention on the same codes, within bounds that follow from
the operator's roundings (kv_ref.attention_bound)."""
import numpy as np
import pytest

import kv_ref as ref
import s3e
from test_zz_no_alloc import _Graphs

pytestmark = pytest.mark.gpu

TYPES = [ref.Q4_0, ref.Q8_0]
FLOAT = {s3e.TYPE_F32: np.float32, s3e.TYPE_F16: np.float16}


def make_cache(ctx, t, heads, D, page, n_pages, rng):
    """A cache of random bytes (what a slot held before must not matter): (cache, its bytes)."""
    c = s3e.KVCache(t, heads, D, page, n_pages)
    mem = rng.integers(0, 256, s3e.kv_cache_bytes(c), dtype=np.uint8)
    return s3e.KVCache(t, heads, D, page, n_pages, ctx.to_device(mem)), mem


def slot_order(rng, order, n, n_pages, page):
    total = n_pages * page
    if order == "scatter":
        return rng.permutation(total)[:n].astype(np.int32)
    if order == "reversed":
        return np.arange(n - 1, -1, -1, dtype=np.int32)
    first = {"aligned": 0, "inside": 5}[order]
    j = np.arange(first, first + n)
    pages = rng.permutation(n_pages)
    return (pages[j // page] * page + j % page).astype(np.int32)


def rows(rng, n, heads, D, io):
    x = rng.standard_normal((n, heads, D)).astype(np.float32) * np.exp(rng.standard_normal((n, 1, 1)))
    return x.astype(FLOAT[io])


WRITES = [
    # t, io, heads, D, page, n, order
    (ref.Q4_0, s3e.TYPE_F32, 1, 32, 32, 1, "inside"),
    (ref.Q4_0, s3e.TYPE_F32, 2, 64, 64, 8, "aligned"),
    (ref.Q4_0, s3e.TYPE_F16, 2, 64, 32, 77, "inside"),
    (ref.Q4_0, s3e.TYPE_F16, 1, 96, 64, 130, "inside"),
    (ref.Q4_0, s3e.TYPE_F32, 3, 128, 128, 71, "aligned"),
    (ref.Q4_0, s3e.TYPE_F16, 1, 256, 256, 69, "inside"),
    (ref.Q4_0, s3e.TYPE_F32, 2, 64, 64, 90, "scatter"),
    (ref.Q4_0, s3e.TYPE_F32, 1, 128, 64, 40, "reversed"),
    (ref.Q8_0, s3e.TYPE_F32, 1, 32, 32, 3, "inside"),
    (ref.Q8_0, s3e.TYPE_F16, 2, 64, 64, 77, "inside"),
    (ref.Q8_0, s3e.TYPE_F32, 1, 96, 32, 66, "aligned"),
    (ref.Q8_0, s3e.TYPE_F16, 2, 128, 128, 50, "scatter"),
    (ref.Q8_0, s3e.TYPE_F32, 1, 256, 64, 70, "inside"),
]


@pytest.mark.parametrize("t,io,heads,D,page,n,order", WRITES)
def test_write_and_read(ctx, t, io, heads, D, page, n, order):
    print(t, io, heads, D, page, n, order, flush=True)
    rng = np.random.default_rng(n * D + heads)
    n_pages = -(-(n + 5) // page) + 1
    c, mem = make_cache(ctx, t, heads, D, page, n_pages, rng)
    slots = slot_order(rng, order, n, n_pages, page)
    if n > 20:  # rows to leave out, in the middle of a run too
        slots[[3, 12]] = [-1, n_pages * page]
    k, v = rows(rng, n, heads, D, io), rows(rng, n, heads, D, io)
    k[0, 0, :32] = 0
    kd, vd, sd = ctx.to_device(k), ctx.to_device(v), ctx.to_device(slots)
    nb = (heads * D, D)
    ctx.kv_write(c, io, kd, nb, vd, nb, sd, n)
    ctx.sync()
    ref.write(mem, t, D, page, heads, slots, k.astype(np.float32), v.astype(np.float32))
    assert np.array_equal(c._data.download(np.uint8, mem.shape), mem)
    for out_io in (s3e.TYPE_F32, s3e.TYPE_F16):
        kb, vb = (ctx.to_device(np.full((n + 1, heads, D), 7, FLOAT[out_io])) for _ in range(2))
        ctx.kv_read(c, sd, n, out_io, kb, vb)
        ctx.sync()
        for x, b in ((k, kb), (v, vb)):
            got = b.download(FLOAT[out_io], (n + 1, heads, D))
            want = ref.values(t, *ref.quantize(t, x.astype(np.float32)))
            want[(slots < 0) | (slots >= n_pages * page)] = 0
            assert np.array_equal(got[:n], want.astype(FLOAT[out_io]))
            assert (got[n] == 7).all()


@pytest.mark.parametrize("t", TYPES)
def test_rows_of_a_fused_projection(ctx, t):
    # strided rows on 4-byte and on 16-byte alignment, and K and V left out of a read
    rng = np.random.default_rng(3)
    heads, D, page, n = 2, 64, 64, 19
    for pad in (0, 1):
        ld = 3 * heads * D + pad
        fused = rng.standard_normal((n, ld)).astype(np.float32)
        c, mem = make_cache(ctx, t, heads, D, page, 2, rng)
        slots = np.arange(7, 7 + n, dtype=np.int32)
        base, sd = ctx.to_device(fused), ctx.to_device(slots)
        at = [s3e.DeviceView(base.ptr + 4 * (i * heads * D + pad), 0) for i in (1, 2)]
        ctx.kv_write(c, s3e.TYPE_F32, at[0], (ld, D), at[1], (ld, D), sd, n)
        k, v = (fused[:, i * heads * D + pad:(i + 1) * heads * D + pad].reshape(n, heads, D) for i in (1, 2))
        ref.write(mem, t, D, page, heads, slots, k, v)
        ctx.sync()
        assert np.array_equal(c._data.download(np.uint8, mem.shape), mem), pad
        out = ctx.to_device(np.zeros((n, heads, D), np.float32))
        ctx.kv_read(c, sd, n, s3e.TYPE_F32, None, out)
        ctx.sync()
        assert np.array_equal(out.download(np.float32, (n, heads, D)), ref.values(t, *ref.quantize(t, v)).astype(np.float32))


@pytest.mark.parametrize("t", TYPES)
def test_unusual_values(ctx, t):
    D, page = 64, 32
    rng = np.random.default_rng(5)
    x = rng.standard_normal((12, 1, D)).astype(np.float32)
    x[0, 0, 5] = np.inf
    x[1, 0, 40] = np.nan
    x[2, 0, 3], x[2, 0, 9] = -9.0, 9.0  # equal magnitudes: the first decides the sign
    x[3, 0, 9], x[3, 0, 17] = 9.0, -9.0
    x[4] = 0
    x[5] = -0.0
    x[6, 0, :32] = 1e30     # a scale past fp16
    x[7] *= np.float32(1e-7)   # fp16 scales that are subnormal or zero
    x[8] *= np.float32(1e-38)
    x[9, 0, :32] = 2.5
    x[10, 0, 31] = 65504.0
    x[11] *= np.float32(1e-42)
    for v in (x, x[::-1].copy()):
        c, mem = make_cache(ctx, t, 1, D, page, 1, rng)
        slots = np.arange(3, 15, dtype=np.int32)
        sd = ctx.to_device(slots)
        ctx.kv_write(c, s3e.TYPE_F32, ctx.to_device(x), (D, D), ctx.to_device(v), (D, D), sd, 12)
        kb, vb = ctx.buffer(x.nbytes), ctx.buffer(x.nbytes)
        ctx.kv_read(c, sd, 12, s3e.TYPE_F32, kb, vb)
        ctx.sync()
        ref.write(mem, t, D, page, 1, slots, x, v)
        assert np.array_equal(c._data.download(np.uint8, mem.shape), mem)
        with np.errstate(all="ignore"):
            for b, y in ((kb, x), (vb, v)):
                want = ref.values(t, *ref.quantize(t, y)).astype(np.float32)
                assert np.array_equal(b.download(np.float32, x.shape), want, equal_nan=True)


def test_matches_the_engines_row_conversion(ctx):
    # Q8_0 codes and scales are s3e_quantize_rows' own
    rng = np.random.default_rng(6)
    n, D = 9, 128
    x = rng.standard_normal((n, 1, D)).astype(np.float32)
    xd = ctx.to_device(x)
    q, d = ctx.buffer(n * D), ctx.buffer(s3e.act_scale_elems(n, D) * 2)
    ctx.quantize_rows(s3e.TYPE_Q8_0, xd, n, D, q, d, None)
    ctx.sync()
    scales = s3e.unstage_scales(d.download(np.uint16, (s3e.act_scale_elems(n, D),)), n, D)
    codes, bits = ref.quantize(ref.Q8_0, x[:, 0])
    assert np.array_equal(q.download(np.int8, (n, D)), codes) and np.array_equal(scales, bits)


def test_slots_far_into_memory(ctx):
    # a cache of 5.3 GB: offsets past 32 bits
    heads, D, page, t = 8, 256, 256, ref.Q4_0
    n_pages = 9000
    c = s3e.KVCache(t, heads, D, page, n_pages)
    size = s3e.kv_cache_bytes(c)
    assert size > 1 << 32
    c = s3e.KVCache(t, heads, D, page, n_pages, ctx.buffer(size))
    rng = np.random.default_rng(9)
    n = 40
    slots = np.concatenate([np.arange(20), n_pages * page - 20 + np.arange(20)]).astype(np.int32)
    k, v = rows(rng, n, heads, D, s3e.TYPE_F16), rows(rng, n, heads, D, s3e.TYPE_F16)
    kd, vd, sd = ctx.to_device(k), ctx.to_device(v), ctx.to_device(slots)
    ctx.kv_write(c, s3e.TYPE_F16, kd, (heads * D, D), vd, (heads * D, D), sd, n)
    kb, vb = ctx.buffer(k.nbytes), ctx.buffer(k.nbytes)
    ctx.kv_read(c, sd, n, s3e.TYPE_F16, kb, vb)
    # a sequence whose last page is the cache's last: its keys are the last 20 slots
    table = np.array([[n_pages - 1]], np.int32)
    q = rows(rng, 1, heads, D, s3e.TYPE_F16)
    len_ = page
    o = ctx.buffer(q.nbytes)
    mask = np.zeros((1, page), np.float16)
    mask[0, :page - 20] = -np.inf  # slots that were never written
    b = s3e.KVBatch(1, 1, 1, len_, ctx.to_device(np.array([0, 1], np.int32)), ctx.to_device(np.array([len_], np.int32)),
                    ctx.to_device(table), 1)
    need = s3e.kv_attn_workspace(c, b, heads, s3e.TYPE_F16)
    ws = ctx.buffer(max(need, 16))
    ctx.kv_attn(c, b, s3e.TYPE_F16, ctx.to_device(q), (heads * D, D), heads, 0.06, o, ws, mask=ctx.to_device(mask), mask_ld=page)
    ctx.sync()
    for x, y in ((k, kb), (v, vb)):
        want = ref.values(t, *ref.quantize(t, x.astype(np.float32))).astype(np.float16)
        assert np.array_equal(y.download(np.float16, k.shape), want)
    parts = [p[20:] for x in (k, v) for p in ref.quantize(t, x.astype(np.float32))]
    want, mag, A = ref.attention(t, *parts, q, 0.06, np.ones((1, 20), bool))
    off = np.abs(o.download(np.float16, q.shape).astype(np.float64) - want)
    assert (off <= ref.attention_bound(False, want, mag, A, 20, D, ref.largest(t, *parts[2:]))).all()


class Batch:
    """Sequences of (queries, keys) in a cache whose other slots, and whose keys' own pages past their end, are random
    bytes; the wanted attention and its bounds."""

    def __init__(self, ctx, t, io, heads, nh, D, page, lens, seed, mask=False, causal=True, max_q=None, max_kv=None,
                 spare_rows=0, pad=0, scale=None, grow=1.0):
        self.ctx, self.t, self.io, self.heads, self.nh, self.D, self.lens = ctx, t, io, heads, nh, D, lens
        rng = np.random.default_rng(seed)
        need = [-(-kv // page) for _, kv in lens]
        n_pages = sum(need) + 2
        self.c, _ = make_cache(ctx, t, heads, D, page, n_pages, rng)
        perm = rng.permutation(n_pages).astype(np.int32)
        ld = max(max(need), 1)
        table = np.full((len(lens), ld), -7, np.int32)
        at, slots, self.kv = 0, [], []
        for i, ((_, kv), n) in enumerate(zip(lens, need)):
            table[i, :n] = perm[at:at + n]
            at += n
            slots += [table[i, j // page] * page + j % page for j in range(kv)]
        n = len(slots)
        self.k = rows(rng, n, heads, D, s3e.TYPE_F32)
        self.v = rows(rng, n, heads, D, s3e.TYPE_F32) * np.float32(grow) ** (np.arange(n) - n * (grow > 1)).astype(np.float32)[:, None, None]
        if n:
            nb = (heads * D, D)
            ctx.kv_write(self.c, s3e.TYPE_F32, ctx.to_device(self.k), nb, ctx.to_device(self.v), nb,
                         ctx.to_device(np.array(slots, np.int32)), n)
        ctx.sync()
        self.starts = np.cumsum([0] + [nq for nq, _ in lens]).astype(np.int32)
        self.n_tokens = int(self.starts[-1]) + spare_rows
        self.ld = nh * D + pad
        self.q = rng.standard_normal((self.n_tokens, self.ld)).astype(FLOAT[io])
        self.max_q = max_q if max_q is not None else max(nq for nq, _ in lens)
        self.max_kv = max_kv if max_kv is not None else max(kv for _, kv in lens)
        self.scale = scale if scale is not None else D ** -0.5
        self.causal, self.mask = causal, None
        if mask:
            m = rng.standard_normal((self.n_tokens, self.max_kv + 3)).astype(np.float16)
            m[rng.random(m.shape) < 0.2] = -np.inf
            m[::5] = -np.inf             # rows that see nothing
            m[1::7] = -65504.0           # rows of the type's lowest value: all keys alike
            self.mask = m
        self.arrays = [ctx.to_device(self.starts), ctx.to_device(np.array([kv for _, kv in lens], np.int32)),
                       ctx.to_device(table)]
        self.b = s3e.KVBatch(len(lens), self.n_tokens, self.max_q, self.max_kv, *self.arrays, ld)
        self.qd = ctx.to_device(self.q)
        self.md = ctx.to_device(self.mask) if mask else None

    def run(self, o=None):
        ctx = self.ctx
        shape = (self.n_tokens, self.nh, self.D)
        o = o or ctx.to_device(np.full(shape, 5, FLOAT[self.io]))
        need = s3e.kv_attn_workspace(self.c, self.b, self.nh, self.io)
        self.ws = ctx.to_device(np.full(need + 16, 0xFF, np.uint8)) if need else None
        ctx.kv_attn(self.c, self.b, self.io, self.qd, (self.ld, self.D), self.nh, self.scale, o, self.ws, causal=self.causal,
                    mask=self.md, mask_ld=self.mask.shape[1] if self.mask is not None else 0)
        ctx.sync()
        return o.download(FLOAT[self.io], shape)

    def want(self):
        at, out = 0, []
        for i, (nq, kv) in enumerate(self.lens):
            parts = [p[at:at + kv] for x in (self.k, self.v) for p in ref.quantize(self.t, x)]
            at += kv
            rows_ = slice(self.starts[i], self.starts[i + 1])
            see = np.arange(kv) <= (kv - nq + np.arange(nq)[:, None]) if self.causal else np.ones((nq, kv), bool)
            see = see & (np.arange(kv) < self.max_kv)
            q = self.q[rows_, :self.nh * self.D].reshape(nq, self.nh, self.D)
            m = self.mask[rows_, :kv] if self.mask is not None else None
            o, mag, A = ref.attention(self.t, *parts, q, self.scale, see, m)
            out.append((o, ref.attention_bound(self.io == s3e.TYPE_F32, o, mag, A, max(kv, 1), self.D, ref.largest(self.t, *parts[2:]))))
        return [np.concatenate(x) for x in zip(*out)]

    def check(self):
        got, (want, bound) = self.run(), self.want()
        n = len(want)
        cut = np.concatenate([np.arange(nq) < self.max_q for nq, _ in self.lens])
        off = np.abs(got[:n].astype(np.float64) - want)
        assert np.isfinite(got[:n]).all()
        assert (off[cut] <= bound[cut]).all(), (off[cut] / bound[cut]).max()
        assert (got[:n][~cut] == 5).all() and (got[n:] == 5).all()
        return got


ATTN = [
    # t, io, heads, nh, D, page, lens, options
    (ref.Q4_0, s3e.TYPE_F32, 1, 1, 32, 32, [(1, 1)], {}),
    (ref.Q4_0, s3e.TYPE_F16, 2, 2, 64, 64, [(1, 77), (1, 0), (1, 31), (1, 33)], {}),
    (ref.Q4_0, s3e.TYPE_F32, 2, 8, 64, 32, [(1, 200), (1, 5)], {}),
    (ref.Q4_0, s3e.TYPE_F16, 1, 5, 96, 64, [(3, 70), (2, 1)], {}),
    (ref.Q4_0, s3e.TYPE_F16, 2, 8, 128, 128, [(1, 1100)], {}),
    (ref.Q4_0, s3e.TYPE_F32, 1, 3, 128, 64, [(7, 300), (7, 4)], {"mask": True}),
    (ref.Q4_0, s3e.TYPE_F16, 2, 2, 64, 64, [(70, 130), (33, 33), (9, 20)], {}),
    (ref.Q4_0, s3e.TYPE_F32, 2, 2, 64, 64, [(70, 130), (33, 10)], {}),
    (ref.Q4_0, s3e.TYPE_F16, 1, 1, 256, 256, [(40, 300)], {"causal": False}),
    (ref.Q4_0, s3e.TYPE_F32, 1, 2, 256, 64, [(20, 90)], {}),
    (ref.Q4_0, s3e.TYPE_F32, 1, 2, 96, 32, [(20, 90), (1, 40)], {"mask": True, "pad": 3}),
    (ref.Q4_0, s3e.TYPE_F16, 1, 2, 32, 32, [(50, 90), (17, 64)], {"mask": True, "pad": 8}),
    (ref.Q8_0, s3e.TYPE_F32, 1, 1, 32, 32, [(1, 3), (1, 64)], {}),
    (ref.Q8_0, s3e.TYPE_F16, 4, 16, 128, 64, [(1, 515), (1, 12)], {}),
    (ref.Q8_0, s3e.TYPE_F32, 2, 8, 128, 64, [(5, 600), (5, 3)], {"mask": True, "causal": False}),
    (ref.Q8_0, s3e.TYPE_F16, 1, 1, 256, 256, [(33, 700)], {"causal": False}),
    (ref.Q8_0, s3e.TYPE_F32, 1, 1, 256, 32, [(18, 60)], {}),
    (ref.Q8_0, s3e.TYPE_F16, 1, 6, 64, 128, [(30, 150), (1, 1)], {"pad": 5}),
    (ref.Q8_0, s3e.TYPE_F32, 2, 4, 96, 64, [(12, 77)], {"spare_rows": 3}),
    (ref.Q8_0, s3e.TYPE_F16, 1, 4, 32, 64, [(9, 44), (3, 44)], {"max_q": 4, "spare_rows": 1}),
    (ref.Q4_0, s3e.TYPE_F16, 1, 2, 64, 64, [(2, 200), (2, 90)], {"max_kv": 128, "causal": False}),
    (ref.Q4_0, s3e.TYPE_F16, 1, 2, 64, 64, [(2, 200)], {"scale": -0.3}),
    (ref.Q8_0, s3e.TYPE_F32, 1, 2, 64, 64, [(2, 200)], {"scale": -0.3}),
    (ref.Q8_0, s3e.TYPE_F16, 1, 2, 64, 64, [(2, 50)], {"scale": 0.0}),
    # V grows by 2^17 over the sequence, or shrinks as far (scales down to fp16's subnormal numbers)
    (ref.Q4_0, s3e.TYPE_F16, 1, 2, 64, 64, [(3, 400)], {"grow": 1.03}),
    (ref.Q8_0, s3e.TYPE_F32, 1, 2, 128, 64, [(3, 400)], {"grow": 1 / 1.03}),
]


@pytest.mark.parametrize("t,io,heads,nh,D,page,lens,more", ATTN)
def test_attention(ctx, t, io, heads, nh, D, page, lens, more):
    print(t, io, heads, nh, D, page, lens, more, flush=True)
    Batch(ctx, t, io, heads, nh, D, page, lens, seed=nh * D + len(lens), **more).check()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("io", [s3e.TYPE_F16, s3e.TYPE_F32])
@pytest.mark.parametrize("D", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("form", ["few", "more", "many", "split"])
def test_every_kernel(ctx, t, io, D, form):
    # up to 16, up to 32 and more columns a key/value head; many columns against several key ranges
    heads, nh, lens, more = {"few": (2, 6, [(3, 300), (2, 33)], {}), "more": (1, 3, [(9, 290), (7, 7)], {"mask": True}),
                             "many": (1, 3, [(90, 300), (37, 37), (50, 12)], {}),
                             "split": (1, 1, [(140, 900)], {"mask": True, "causal": False})}[form]
    print(t, io, D, form, flush=True)
    x = Batch(ctx, t, io, heads, nh, D, 64, lens, seed=D + len(form), **more)
    assert form != "split" or s3e.kv_attn_workspace(x.c, x.b, nh, io) > 0
    x.check()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("io", [s3e.TYPE_F16, s3e.TYPE_F32])
@pytest.mark.parametrize("D,nq", [(64, 2), (64, 20), (64, 70), (128, 70), (256, 40)])
def test_a_key_hidden_from_some_queries(ctx, t, io, D, nq):
    # its NaN reaches the queries that see it and no others, though lanes hold columns of both kinds
    kv = 100
    x = Batch(ctx, t, io, 1, 1, D, 64, [(nq, kv)], seed=nq, mask=True, causal=False)
    x.mask[:] = 0
    x.mask[::2, 33] = -np.inf
    x.mask[1::3, 70:80] = -np.inf
    x.md.upload(x.mask)
    table = x.arrays[2].download(np.int32, (1, 2))
    slots = np.array([table[0, j // 64] * 64 + j % 64 for j in range(kv)], np.int32)
    k, v = x.k.copy(), x.v.copy()
    v[33] = np.nan
    ctx.kv_write(x.c, s3e.TYPE_F32, ctx.to_device(k), (D, D), ctx.to_device(v), (D, D), ctx.to_device(slots), kv)
    got = x.run()
    want, bound = x.want()  # (of the rows that do not see key 33: its value has no part in them)
    assert np.isnan(got[1::2]).all()
    assert (np.abs(got[::2].astype(np.float64) - want[::2]) <= bound[::2]).all()


@pytest.mark.parametrize("t", TYPES)
def test_pairs_are_whole(ctx, t):
    # the high half of every fp32 pair is the one its low half completes: 40 x 10^4 products a call, ties among them
    for seed in range(6):
        Batch(ctx, t, s3e.TYPE_F32, 2, 4, 64, 32, [(45, 45), (7, 7)], seed=seed).check()


@pytest.mark.parametrize("io", [s3e.TYPE_F16, s3e.TYPE_F32])
def test_attention_writes_in_place(ctx, io):
    x = Batch(ctx, ref.Q4_0, io, 2, 4, 64, 64, [(5, 700), (2, 90)], seed=4)
    apart = x.check()
    assert np.array_equal(x.run(o=x.qd), apart)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("io", [s3e.TYPE_F16, s3e.TYPE_F32])
def test_hidden_keys_reach_nothing(ctx, t, io):
    # NaN and infinite K and V in masked places, keys past the end and a page that the cache does not have
    heads, nh, D, page, kv = 1, 2, 64, 32, 150
    x = Batch(ctx, t, io, heads, nh, D, page, [(2, kv)], seed=8, mask=True, causal=False)
    x.mask[:] = 0
    x.mask[:, 10:20] = -np.inf
    x.mask[:, 64:96] = -np.inf
    x.md.upload(x.mask)
    x.k[10:20], x.v[10:20] = np.nan, np.inf
    x.k[15], x.v[15] = 1e30, 1e30
    table = x.arrays[2].download(np.int32, (1, 5))
    slots = np.array([table[0, j // page] * page + j % page for j in range(kv)], np.int32)
    nb = (heads * D, D)
    ctx.kv_write(x.c, s3e.TYPE_F32, ctx.to_device(x.k), nb, ctx.to_device(x.v), nb, ctx.to_device(slots), kv)
    for page_id in (table[0, 2], -1, 1 << 30):
        table[0, 2] = page_id
        x.arrays[2].upload(table)
        x.check()
    # the same keys hidden by the page alone
    x.mask[:, 64:96] = 0
    x.md.upload(x.mask)
    got = x.run()
    x.mask[:, 64:96] = -np.inf
    x.md.upload(x.mask)
    assert np.array_equal(x.run(), got)


@pytest.mark.parametrize("io", [s3e.TYPE_F16, s3e.TYPE_F32])
@pytest.mark.parametrize("t", [ref.Q4_0, ref.Q8_0])
@pytest.mark.parametrize("nq", [3, 40])
@pytest.mark.parametrize("masked", [False, True])
def test_large_hidden_values_change_nothing(ctx, t, io, nq, masked):
    # keys that a row does not see (later ones, or masked ones) with values near the largest a cache holds, among
    # small ones: the row's bits are those beside small keys.  nq: one or more column tiles
    heads, nh, D, page, kv = 1, 2, 64, 64, 120
    x = Batch(ctx, t, io, heads, nh, D, page, [(nq, kv)], seed=21, mask=masked, causal=not masked)
    hide = np.arange(kv) >= kv - nq // 2 if not masked else np.arange(kv) % 9 == 4
    rows = np.arange(nq) < nq - nq // 2 if not masked else np.ones(nq, bool)
    if masked:
        x.mask[:, :kv] = np.where(hide, -np.inf, 0)
        x.md.upload(x.mask)
    table = x.arrays[2].download(np.int32, (1, -(-kv // page)))
    slots = ctx.to_device(np.array([table[0, j // page] * page + j % page for j in range(kv)], np.int32))
    nb = (heads * D, D)
    outs = []
    for large in (1e-3, 1e5):
        k, v = x.k * 1.0, x.v * 1e-3
        v[hide] *= large / 1e-3
        ctx.kv_write(x.c, s3e.TYPE_F32, ctx.to_device(k.astype(np.float32)), nb, ctx.to_device(v.astype(np.float32)), nb, slots, kv)
        outs.append(x.run()[rows])
    assert np.isfinite(outs[0]).all() and np.abs(outs[0]).max() > 0
    assert np.array_equal(outs[0], outs[1])


@pytest.mark.parametrize("io", [s3e.TYPE_F16, s3e.TYPE_F32])
def test_values_that_are_no_numbers_come_through(ctx, io):
    x = Batch(ctx, ref.Q8_0, io, 1, 1, 64, 64, [(1, 90), (1, 40)], seed=2)
    x.v[3, 0, 0] = np.nan    # the first block of key 3 of the first sequence
    x.k[90 + 2, 0, 40] = np.nan  # a score of the second
    table = x.arrays[2].download(np.int32, (2, 2))
    slots = np.array([table[0, j // 64] * 64 + j % 64 for j in range(90)] + [table[1, 0] * 64 + j for j in range(40)], np.int32)
    ctx.kv_write(x.c, s3e.TYPE_F32, ctx.to_device(x.k), (64, 64), ctx.to_device(x.v), (64, 64), ctx.to_device(slots), 130)
    got = x.run()
    assert np.isnan(got[0, 0, :32]).all() and np.isfinite(got[0, 0, 32:]).all()
    assert np.isnan(got[1]).all()


@pytest.mark.parametrize("magnitude", [1e-30, 1e-3, 1e4, 1e30])
def test_f32_queries_of_any_magnitude(ctx, magnitude):
    x = Batch(ctx, ref.Q8_0, s3e.TYPE_F32, 1, 2, 64, 64, [(3, 100)], seed=11, scale=float(np.float32(0.125 / magnitude)))
    x.q *= np.float32(magnitude)
    x.qd.upload(x.q)
    x.check()


def test_repeated_calls_are_identical(ctx):
    x = Batch(ctx, ref.Q4_0, s3e.TYPE_F16, 2, 8, 128, 64, [(1, 3000), (1, 10)], seed=12)
    first = x.check()
    for _ in range(3):
        assert np.array_equal(x.run(), first)


@pytest.mark.parametrize("io", [s3e.TYPE_F16, s3e.TYPE_F32])
def test_captured_decoding(ctx, io):
    """One captured step (write the new token, attend) replayed while lengths grow, beside eager work; and two graphs
    with workspaces of their own on two streams at once."""
    import ctypes

    heads, nh, D, page, t = 2, 4, 64, 32, ref.Q4_0
    rng = np.random.default_rng(21)
    gr = _Graphs()
    gr.h.hipStreamCreateWithFlags.argtypes = [ctypes.POINTER(ctypes.c_void_p), ctypes.c_uint]
    gr.h.hipStreamSynchronize.argtypes = gr.h.hipStreamDestroy.argtypes = [ctypes.c_void_p]
    other = ctypes.c_void_p()
    assert gr.h.hipStreamCreateWithFlags(ctypes.byref(other), 1) == 0
    steps, most = 6, 1500
    seqs = []
    for i in range(2):
        x = Batch(ctx, t, io, heads, nh, D, page, [(1, most)], seed=30 + i)
        table = x.arrays[2].download(np.int32, (1, -(-most // page)))
        slots = np.array([table[0, j // page] * page + j % page for j in range(most)], np.int32)
        new = dict(k=ctx.buffer(heads * D * 4), v=ctx.buffer(heads * D * 4), slot=ctx.buffer(4))
        need = s3e.kv_attn_workspace(x.c, x.b, nh, io)
        assert need > 0
        ws, o = ctx.buffer(need), ctx.buffer(x.q.nbytes)

        def step(x=x, new=new, ws=ws, o=o):
            ctx.kv_write(x.c, s3e.TYPE_F32, new["k"], (heads * D, D), new["v"], (heads * D, D), new["slot"], 1)
            ctx.kv_attn(x.c, x.b, io, x.qd, (x.ld, D), nh, x.scale, o, ws, causal=True)

        new["slot"].upload(np.array([-1], np.int32))
        step()
        ctx.sync()
        seqs.append((x, slots, new, o, gr.capture(ctx.stream, step)))
    try:
        for s in range(steps):
            kv = [200 + 211 * s, most - 97 * s]
            for (x, slots, new, o, _), n in zip(seqs, kv):
                x.k[n - 1], x.v[n - 1] = rng.standard_normal((heads, D)), rng.standard_normal((heads, D))
                new["k"].upload(x.k[n - 1])
                new["v"].upload(x.v[n - 1])
                new["slot"].upload(slots[n - 1:n])
                x.arrays[1].upload(np.array([n], np.int32))
                o.upload(np.full((1, nh, D), np.nan, FLOAT[io]))
            for (_, _, _, _, (_, ex)), st in zip(seqs, (ctx.stream, other)):
                assert gr.h.hipGraphLaunch(ex, st) == 0
            ctx.sync()
            assert gr.h.hipStreamSynchronize(other) == 0
            for (x, slots, new, o, _), n in zip(seqs, kv):
                got = o.download(FLOAT[io], (1, nh, D))
                assert np.array_equal(x.run(), got), s  # the same call made eagerly, between the replays
                parts = [p[:n] for y in (x.k, x.v) for p in ref.quantize(t, y)]
                w, mag, A = ref.attention(t, *parts, x.q.reshape(1, nh, D), x.scale, np.ones((1, n), bool))
                off = np.abs(got.astype(np.float64) - w)
                assert (off <= ref.attention_bound(io == s3e.TYPE_F32, w, mag, A, n, D, ref.largest(t, *parts[2:]))).all(), s
    finally:
        for _, _, _, _, (g, ex) in seqs:
            gr.h.hipGraphExecDestroy(ex)
            gr.h.hipGraphDestroy(g)
        gr.h.hipStreamDestroy(other)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("io", [s3e.TYPE_F16, s3e.TYPE_F32])
@pytest.mark.parametrize("kv", [20, 33, 65, 97, 700])
def test_many_columns_of_256(ctx, t, io, kv):
    # the kernel for many columns at head dim 256: odd and even numbers of chunks, one of them, several key ranges,
    # a last work-group with few columns, rows that see nothing
    Batch(ctx, t, io, 1, 2, 256, 32, [(150, kv)], seed=kv).check()
    Batch(ctx, t, io, 1, 2, 256, 64, [(3, 5), (131, kv)], seed=kv, mask=True, causal=False).check()


@pytest.mark.parametrize("t", TYPES)
def test_a_key_hidden_from_some_of_many_columns(ctx, t):
    kv, nq, D = 100, 300, 256
    x = Batch(ctx, t, s3e.TYPE_F16, 1, 1, D, 64, [(nq, kv)], seed=nq, mask=True, causal=False)
    x.mask[:] = 0
    x.mask[::2, 33] = -np.inf
    x.md.upload(x.mask)
    table = x.arrays[2].download(np.int32, (1, 2))
    slots = np.array([table[0, j // 64] * 64 + j % 64 for j in range(kv)], np.int32)
    v = x.v.copy()
    v[33] = np.nan
    ctx.kv_write(x.c, s3e.TYPE_F32, ctx.to_device(x.k), (D, D), ctx.to_device(v), (D, D), ctx.to_device(slots), kv)
    got = x.run()
    want, bound = x.want()
    assert np.isnan(got[1::2]).all()
    assert (np.abs(got[::2].astype(np.float64) - want[::2]) <= bound[::2]).all()


@pytest.mark.parametrize("io", [s3e.TYPE_F16, s3e.TYPE_F32])
@pytest.mark.parametrize("nq", [1, 20])
def test_many_sequences(ctx, io, nq):
    # 203 of them, some without queries, some without keys, in a number that no XCD's share divides
    rng = np.random.default_rng(nq)
    lens = [(int(rng.integers(0, nq + 1)), int(rng.integers(0, 80))) for _ in range(203)]
    Batch(ctx, ref.Q4_0, io, 1, 3, 32, 32, lens, seed=5, max_q=nq).check()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("io", [s3e.TYPE_F16, s3e.TYPE_F32])
def test_writers_of_neighbouring_slots_at_once(ctx, t, io):
    # two contexts write every other slot, so that each word of V holds codes of both, and runs beside lone rows
    rng = np.random.default_rng(31)
    heads, D, page, n_pages = 2, 96, 64, 5
    n = n_pages * page // 2
    other = s3e.Context()
    c, mem = make_cache(ctx, t, heads, D, page, n_pages, rng)
    nb = (heads * D, D)
    calls = []
    for cx, slots in ((ctx, np.arange(0, 2 * n, 2)), (other, np.arange(1, 2 * n, 2))):
        slots = slots.astype(np.int32)
        if cx is ctx:
            slots = rng.permutation(slots)
        k, v = rows(rng, n, heads, D, io), rows(rng, n, heads, D, io)
        ref.write(mem, t, D, page, heads, slots, k.astype(np.float32), v.astype(np.float32))
        calls.append((cx, cx.to_device(k), cx.to_device(v), cx.to_device(slots)))
    for cx, _, _, _ in calls:
        cx.sync()
    for _ in range(3):
        for cx, kd, vd, sd in calls:
            cx.kv_write(c, io, kd, nb, vd, nb, sd, n)
    for cx, _, _, _ in calls:
        cx.sync()
    assert np.array_equal(c._data.download(np.uint8, mem.shape), mem)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("lone", [False, True])
def test_a_slot_given_twice_harms_no_other(ctx, t, lone):
    rng = np.random.default_rng(8)
    heads, D, page = 2, 64, 32
    c, mem = make_cache(ctx, t, heads, D, page, 3, rng)
    # slot 5 twice: among scattered rows, or in a run of eight and again behind it
    slots = np.array([5, 40, 70, 5, 2, 3] if lone else list(range(8, 16)) + list(range(0, 8)) + [5], np.int32)
    n = len(slots)
    k, v = rows(rng, n, heads, D, s3e.TYPE_F32), rows(rng, n, heads, D, s3e.TYPE_F32)
    nb = (heads * D, D)
    ctx.kv_write(c, s3e.TYPE_F32, ctx.to_device(k), nb, ctx.to_device(v), nb, ctx.to_device(slots), n)
    ctx.sync()
    got = c._data.download(np.uint8, mem.shape)
    ref.write(mem, t, D, page, heads, slots, k, v)
    # whatever slot 5 holds, write it again on both sides
    again = np.array([5], np.int32)
    c._data.upload(got)
    ctx.kv_write(c, s3e.TYPE_F32, ctx.to_device(k[:1]), nb, ctx.to_device(v[:1]), nb, ctx.to_device(again), 1)
    ctx.sync()
    ref.write(mem, t, D, page, heads, again, k[:1], v[:1])
    assert np.array_equal(c._data.download(np.uint8, mem.shape), mem)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("D", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("nq,kv", [(1, 2), (1, 128), (7, 40), (30, 128)])
def test_few_keys_in_fp16_round_once(ctx, t, D, nq, kv):
    # up to 128 keys: the products with V's scales are pairs as in fp32, and the output's rounding to fp16 (2^-11, and
    # 2^-25 below its normal numbers) is all that is added to fp32's bound
    x = Batch(ctx, t, s3e.TYPE_F16, 1, 2, D, 64, [(nq, kv), (nq, nq)], seed=D + kv, max_kv=max(kv, nq))
    got = x.run().astype(np.float64)
    at = 0
    for i, (n, keys) in enumerate(x.lens):
        parts = [p[at:at + keys] for y in (x.k, x.v) for p in ref.quantize(t, y)]
        at += keys
        see = np.arange(keys) <= (keys - n + np.arange(n)[:, None])
        q = x.q[x.starts[i]:x.starts[i + 1], :2 * D].reshape(n, 2, D)
        o, mag, A = ref.attention(t, *parts, q, x.scale, see)
        bound = ref.attention_bound(True, o, mag, A, keys, D, ref.largest(t, *parts[2:]))
        assert (np.abs(got[x.starts[i]:x.starts[i + 1]] - o) <= bound * (1 + 2.0 ** -11) + np.abs(o) * 2.0 ** -11 + 2.0 ** -25).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("io", [s3e.TYPE_F16, s3e.TYPE_F32])
@pytest.mark.parametrize("D", [32, 128, 256])
@pytest.mark.parametrize("at", [0, 4, 9])
def test_a_prompt_among_single_tokens(ctx, t, io, D, at):
    # work-groups that look their sequence up: the prompt first, inside or last, sequences without rows or keys, several
    # key ranges, more rows than the sequences have
    tokens = [(1, 90), (1, 3), (0, 40), (1, 1000), (2, 2), (1, 0), (0, 0), (1, 31), (1, 257)]
    lens = tokens[:at] + [(130, 200)] + tokens[at:]
    for heads, nh, more in ((1, 3, {}), (8, 8, {"spare_rows": 5, "mask": True, "causal": False})):
        Batch(ctx, t, io, heads, nh, D, 64, lens, seed=at + D, **more).check()


@pytest.mark.parametrize("io", [s3e.TYPE_F16, s3e.TYPE_F32])
@pytest.mark.parametrize("D", [64, 96])
def test_a_prompt_beside_a_long_token(ctx, io, D):
    # many key ranges, joined row by row where the bounds hold far more rows than there are
    x = Batch(ctx, ref.Q4_0, io, 1, 2, D, 64, [(1, 10), (33, 300), (0, 50), (1, 4000), (1, 0)], seed=D, spare_rows=2)
    assert s3e.kv_attn_workspace(x.c, x.b, 2, io) > 8 * x.n_tokens * 2 * (D + 2) * 4
    x.check()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("io", [s3e.TYPE_F16, s3e.TYPE_F32])
@pytest.mark.parametrize("D,lens", [(64, [(2, 200), (5, 130), (1, 100)]), (128, [(40, 150), (3, 128), (1, 900)]),
                                    (256, [(150, 200), (150, 140)]), (64, [(1, 300), (1, 20), (70, 190), (1, 129), (1, 131)])])
def test_causal_rows_of_sequences_longer_than_max_kv(ctx, t, io, D, lens):
    # row i of nq sees keys up to kv_len - nq + i, cut at max_kv: not up to max_kv - nq + i
    Batch(ctx, t, io, 1, 2, D, 64, lens, seed=D, max_kv=128).check()


def few_keys_bound(o, bound, visible):
    """A bound for fp16 rows by the keys that they see (their sequence's length and the causal limit): up to 128 of them
    fp32's, and the output's rounding to fp16 (2^-11, and 2^-25 below its normal numbers)."""
    few = visible <= 128
    return few, bound * (1 + 2.0 ** -11) + np.abs(o) * 2.0 ** -11 + 2.0 ** -25


def check_few_keys(x, n_checked):
    got, at, checked = x.run().astype(np.float64), 0, 0
    for i, (n, keys) in enumerate(x.lens):
        parts = [p[at:at + keys] for y in (x.k, x.v) for p in ref.quantize(x.t, y)]
        at += keys
        see = np.arange(keys) <= (keys - n + np.arange(n)[:, None]) if x.causal else np.ones((n, keys), bool)
        rows_ = slice(x.starts[i], x.starts[i + 1])
        q = x.q[rows_, :x.nh * x.D].reshape(n, x.nh, x.D)
        o, mag, A = ref.attention(x.t, *parts, q, x.scale, see)
        few, bound = few_keys_bound(o, ref.attention_bound(True, o, mag, A, keys, x.D, ref.largest(x.t, *parts[2:])), see.sum(-1))
        off = np.abs(got[rows_] - o)
        assert (off[few] <= bound[few]).all(), (i, (off[few] / bound[few]).max())
        checked += few.sum()
    assert checked == n_checked


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("nq,kv,causal", [(100, 128, True), (300, 128, False), (300, 40, False)])
def test_many_columns_of_few_keys_round_once(ctx, t, nq, kv, causal):
    # head dim 256, more columns than one work-group of the other kernel takes.  (A small scale: the bound of the scores'
    # own roundings, 2^-24 · (D + 8) · their size, would hide one of P·d at this head dim)
    x = Batch(ctx, t, s3e.TYPE_F16, 1, 1, 256, 64, [(nq, kv)], seed=nq + kv, causal=causal, scale=1e-4)
    check_few_keys(x, nq)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("D,lens,causal", [
    (64, [(1, 20), (1, 2000), (1, 128)], True), (128, [(5, 40), (3, 1000), (2, 129)], False), (96, [(30, 100), (30, 30), (7, 700)], True),
    (32, [(200, 200)], True), (128, [(140, 300)], True), (64, [(150, 180), (150, 150)], True),
    (256, [(1, 20), (1, 2000)], True), (256, [(300, 300), (40, 60)], True), (256, [(300, 90), (3, 500)], False),
    (64, [(130, 130), (1, 5), (1, 900), (1, 0), (1, 60)], True)])
def test_rows_of_few_keys_round_once_in_any_batch(ctx, t, D, lens, causal):
    # whatever the batch's bounds, and the later rows of a prompt, are: the first rows of a prompt and short sequences
    # (heads: of one and of three columns a query; more sequences than the bounds need, so that one finds its own)
    for heads, nh in ((1, 1), (2, 6)):
        x = Batch(ctx, t, s3e.TYPE_F16, heads, nh, D, 64, lens, seed=D + nh, causal=causal, scale=1e-4, spare_rows=1)
        check_few_keys(x, sum(int((np.minimum(kv, kv - nq + np.arange(nq) + 1) <= 128).sum()) if causal else nq * (kv <= 128) for nq, kv in lens))
        assert (x.run()[x.starts[-1]:] == 5).all()


IN_PLACE = [
    # t, heads, nh, D, lens, causal: one range of keys, so that the attention kernel itself stores over q; several column
    # tiles of a sequence, rows that see no key, sequences without keys, grouped heads
    (ref.Q4_0, 1, 1, 64, [(70, 200), (3, 2), (1, 0)], True), (ref.Q8_0, 2, 6, 64, [(70, 100), (33, 33)], False),
    (ref.Q8_0, 1, 3, 128, [(50, 20), (1, 7)], True), (ref.Q4_0, 2, 4, 32, [(1, 90), (1, 0), (1, 250)], True),
    # the kernel for many columns at head dim 256: a last work-group with waves that hold no column
    (ref.Q8_0, 1, 1, 256, [(150, 200)], False), (ref.Q8_0, 1, 2, 256, [(110, 20), (140, 240)], True),
    (ref.Q4_0, 1, 1, 256, [(300, 200), (5, 0)], True), (ref.Q8_0, 1, 1, 256, [(200, 0), (1, 3)], True)]


@pytest.mark.parametrize("io", [s3e.TYPE_F16, s3e.TYPE_F32])
@pytest.mark.parametrize("t,heads,nh,D,lens,causal", IN_PLACE)
def test_attention_in_one_range_writes_in_place(ctx, io, t, heads, nh, D, lens, causal):
    x = Batch(ctx, t, io, heads, nh, D, 64, lens, seed=len(lens) + D, causal=causal)
    assert s3e.kv_attn_workspace(x.c, x.b, nh, io) == 0
    apart = x.check()
    for _ in range(3):
        x.qd.upload(x.q)
        assert np.array_equal(x.run(o=x.qd), apart)


@pytest.mark.parametrize("io", [s3e.TYPE_F16, s3e.TYPE_F32])
@pytest.mark.parametrize("scale", [3.4e38, -3.4e38, 1e-45])
def test_scales_at_the_ends_of_fp32(ctx, io, scale):
    # queries of zeros: every score is zero, whatever the finite scale, and the output V's mean
    x = Batch(ctx, ref.Q8_0, io, 1, 2, 64, 64, [(3, 100), (20, 40)], seed=4, scale=scale, causal=False)
    x.q[:] = 0
    x.qd.upload(x.q)
    x.check()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("io", [s3e.TYPE_F16, s3e.TYPE_F32])
@pytest.mark.parametrize("D,nq,kv", [(64, 3, 90), (128, 40, 300), (256, 150, 200)])
def test_channel_blocks_of_unlike_size(ctx, t, io, D, nq, kv):
    # V's first 32 channels 2^10 times the others, every other key 2^6 times its neighbour: the bound's 2^-31 of the
    # largest |V| a key is what small blocks and small keys are held to
    x = Batch(ctx, t, io, 1, 2, D, 64, [(nq, kv)], seed=D + nq)
    x.v *= np.float32(2.0 ** -6)
    x.v[:, :, 32:] *= np.float32(2.0 ** -10)
    x.v[::2] *= np.float32(2.0 ** 6)
    table = x.arrays[2].download(np.int32, (1, -(-kv // 64)))
    slots = np.array([table[0, j // 64] * 64 + j % 64 for j in range(kv)], np.int32)
    ctx.kv_write(x.c, s3e.TYPE_F32, ctx.to_device(x.k), (D, D), ctx.to_device(x.v), (D, D), ctx.to_device(slots), kv)
    x.check()
