"""What the quantized key/value cache's entry points refuse, without a GPU:
every check is made before anything reaches the device."""
import ctypes

import numpy as np
import pytest

import s3e

# any address: a refused call reads no memory, and no call here is accepted with work to do
FAKE = 1 << 20
CTX = ctypes.cast(ctypes.create_string_buffer(4096), ctypes.c_void_p)


class Buf:
    def __init__(self, ptr=FAKE, nbytes=1 << 40):
        self.ptr, self.nbytes = ptr, nbytes


def cache(**over):
    a = dict(ggml_type=s3e.TYPE_Q4_0, n_heads=2, head_dim=64, page=64, n_pages=4, data=Buf())
    a.update(over)
    return s3e.KVCache(**a)


def batch(**over):
    a = dict(n_seq=2, n_tokens=6, max_q=3, max_kv=200, q_start=Buf(), kv_len=Buf(), pages=Buf(), pages_ld=4)
    a.update(over)
    return s3e.KVBatch(**a)


def write(c, n=3, type_=s3e.TYPE_F32, k=FAKE, v=FAKE, k_nb=(128, 64), v_nb=(128, 64), slots=FAKE, ctx=CTX):
    return s3e.LIB.s3e_kv_write(ctx, ctypes.byref(c) if c else None, type_, k, (ctypes.c_int64 * 2)(*k_nb), v,
                                (ctypes.c_int64 * 2)(*v_nb), slots, n)


def read(c, n=3, type_=s3e.TYPE_F32, k=FAKE, v=FAKE, slots=FAKE, ctx=CTX):
    return s3e.LIB.s3e_kv_read(ctx, ctypes.byref(c) if c else None, slots, n, type_, k, v)


O, WS = FAKE + (1 << 28), FAKE + (1 << 30)


def attn(c=None, b=None, type_=s3e.TYPE_F32, q=FAKE + (1 << 24), q_nb=(256, 64), nh=4, scale=0.125, mask=None, mask_ld=0,
         o=O, ws=WS, ws_bytes=1 << 40, ctx=CTX):
    c, b = c or cache(), b or batch()
    return s3e.LIB.s3e_kv_attn(ctx, ctypes.byref(c), ctypes.byref(b), type_, q, (ctypes.c_int64 * 2)(*q_nb), nh, scale, 0,
                               mask, mask_ld, o, ws, ws_bytes)


INVALID, UNSUPPORTED = 1, 4

BAD_CACHES = [
    (dict(ggml_type=s3e.TYPE_F16), UNSUPPORTED), (dict(ggml_type=s3e.TYPE_Q4_1), UNSUPPORTED),
    (dict(head_dim=48), UNSUPPORTED), (dict(head_dim=0), UNSUPPORTED), (dict(head_dim=160), UNSUPPORTED),
    (dict(page=16), UNSUPPORTED), (dict(page=48), UNSUPPORTED), (dict(n_heads=0), INVALID), (dict(n_heads=-1), INVALID),
    (dict(n_pages=0), INVALID), (dict(n_pages=1 << 26), INVALID), (dict(data=Buf(FAKE + 8)), INVALID),
]


@pytest.mark.parametrize("over,status", BAD_CACHES)
def test_bad_cache(over, status):
    c = cache(**over)
    n = ctypes.c_size_t()
    assert s3e.LIB.s3e_kv_cache_bytes(ctypes.byref(c), ctypes.byref(n)) == status
    assert write(c) == status and read(c) == status and attn(c) == status
    assert s3e.LIB.s3e_last_error()


def test_cache_bytes():
    # 2 heads · 256 slots · 64 channels, K and V: 18 / 34 bytes a block of 32
    assert s3e.kv_cache_bytes(cache()) == 2 * 2 * 256 * 2 * 18
    assert s3e.kv_cache_bytes(cache(ggml_type=s3e.TYPE_Q8_0, data=None)) == 2 * 2 * 256 * 2 * 34
    # past 32 bits
    assert s3e.kv_cache_bytes(cache(n_pages=1 << 24, head_dim=128, n_heads=8)) == (1 << 30) * 8 * 128 // 8 * 9


def test_bad_rows():
    c = cache()
    assert write(None) == INVALID and read(None) == INVALID
    assert write(c, ctx=None) == INVALID and read(c, ctx=None) == INVALID
    for over in (dict(k=None), dict(v=None), dict(slots=None), dict(n=-1), dict(n=1 << 31), dict(k_nb=(-128, 64)),
                 dict(v_nb=(128, -1)), dict(k=FAKE + 2), dict(v=FAKE + 1, type_=s3e.TYPE_F16)):
        assert write(c, **over) == INVALID, over
    for over in (dict(k=None, v=None), dict(slots=None), dict(n=-1), dict(n=1 << 31), dict(k=FAKE + 8), dict(v=FAKE + 4)):
        assert read(c, **over) == INVALID, over
    assert write(c, type_=s3e.TYPE_Q4_0) == UNSUPPORTED and read(c, type_=3) == UNSUPPORTED
    assert write(cache(data=None)) == INVALID and read(cache(data=None)) == INVALID


def test_nothing_to_do_succeeds():
    assert write(cache(), n=0) == 0 and read(cache(), n=0) == 0
    for over in (dict(n_seq=0), dict(n_tokens=0), dict(max_q=0)):
        assert attn(b=batch(**over)) == 0, over
        assert s3e.kv_attn_workspace(cache(), batch(**over), 4, s3e.TYPE_F16) == 0


def test_bad_batches():
    for over in (dict(n_seq=-1), dict(n_seq=65536), dict(n_tokens=-1), dict(max_q=-1), dict(max_kv=-1), dict(pages_ld=-1),
                 dict(max_kv=257), dict(max_kv=1 << 40, pages_ld=1 << 36), dict(n_tokens=1 << 31), dict(max_q=1 << 30)):
        b = batch(**over)
        assert attn(b=b) == INVALID, over
        n = ctypes.c_size_t()
        assert s3e.LIB.s3e_kv_attn_workspace(ctypes.byref(cache()), ctypes.byref(b), 4, 0, ctypes.byref(n)) == INVALID, over
    for name in ("q_start", "kv_len", "pages"):
        assert attn(b=batch(**{name: None})) == INVALID, name
    for nh in (0, 3, -2, 1 << 17):
        assert attn(nh=nh) == INVALID, nh


def test_bad_attention_arguments():
    for over in (dict(q=None), dict(o=None), dict(ctx=None), dict(q_nb=(-256, 64)), dict(q=FAKE + 2), dict(o=O + 8),
                 dict(scale=float("nan")), dict(scale=float("inf")), dict(mask=FAKE, mask_ld=199), dict(mask=FAKE + 1, mask_ld=256),
                 dict(o=FAKE + (1 << 24) + 64), dict(o=FAKE)):
        assert attn(**over) == INVALID, over
    assert attn(type_=s3e.TYPE_Q8_0) == UNSUPPORTED


def test_overlaps_are_refused():
    c = cache()
    nb = s3e.kv_cache_bytes(c)
    far = FAKE + (1 << 30)
    ok = dict(k=far, v=far, slots=far + (1 << 20))  # (k and v may be the same rows)
    # the last row of k or v, or the slots, run into the cache: three rows of two heads of 64 floats
    for over in (dict(k=FAKE - 1532), dict(v=FAKE + nb - 4), dict(slots=FAKE - 8)):
        assert write(c, **{**ok, **over}) == INVALID, over
        assert b"overlap" in s3e.LIB.s3e_last_error()
    ok = dict(k=far, v=far + 3 * 512, slots=far + (1 << 20))
    for over in (dict(v=far + 3 * 512 - 16), dict(k=FAKE - 1520), dict(v=FAKE + nb - 16), dict(slots=far + 1024), dict(k=None, slots=far + 3 * 512)):
        assert read(c, **{**ok, **over}) == INVALID, over
        assert b"overlap" in s3e.LIB.s3e_last_error()
    # the output of attention: six rows of four heads of 64 floats
    ob = 6 * 4 * 64 * 4
    for over in (dict(mask=O + ob - 2, mask_ld=256), dict(mask=O - 16, mask_ld=200)):
        assert attn(**over) == INVALID, over
        assert b"overlap" in s3e.LIB.s3e_last_error()
    for name in ("q_start", "kv_len", "pages"):
        assert attn(b=batch(**{name: Buf(O + ob - 4)})) == INVALID, name
        assert b"overlap" in s3e.LIB.s3e_last_error()
    # the workspace
    b = dict(n_seq=1, n_tokens=1, max_q=1, max_kv=100000, pages_ld=2000)
    c = cache(n_pages=2000)
    far = FAKE + (1 << 36)
    for name in ("q_start", "kv_len", "pages"):
        assert attn(c, batch(**b, **{name: Buf(WS + 64)}), o=far) == INVALID, name
        assert b"overlap" in s3e.LIB.s3e_last_error()
    assert attn(c, batch(**b), o=far, mask=WS + 64, mask_ld=100000) == INVALID
    assert b"overlap" in s3e.LIB.s3e_last_error()


def test_strides_past_any_memory_are_refused():
    far = FAKE + (1 << 30)
    for nb in ((1 << 62, 64), (128, 1 << 62), (1 << 60, 64)):
        assert write(cache(), k=far, v=far, k_nb=nb) == INVALID and b"strides" in s3e.LIB.s3e_last_error(), nb
        assert attn(q_nb=nb) == INVALID and b"strides" in s3e.LIB.s3e_last_error(), nb
    assert attn(mask=far, mask_ld=1 << 61) == INVALID and b"mask" in s3e.LIB.s3e_last_error()
    assert write(cache(), n=(1 << 29) + 1) == INVALID and read(cache(), n=(1 << 29) + 1) == INVALID


def test_workspace_is_checked():
    # one long sequence: its keys go in ranges, whose partial results need memory
    b = batch(n_seq=1, n_tokens=1, max_q=1, max_kv=100000, pages_ld=2000)
    need = s3e.kv_attn_workspace(cache(n_pages=2000), b, 4, s3e.TYPE_F16)
    assert need > 0 and need % (4 * 66 * 4) == 0  # ranges of [1][4 heads][64 + 2] floats
    c = cache(n_pages=2000)
    far = FAKE + (1 << 36)
    assert attn(c, b, ws=None, o=far) == INVALID and attn(c, b, ws_bytes=need - 1, o=far) == INVALID
    assert attn(c, b, ws=WS + 4, o=far) == INVALID
    assert attn(c, b, ws=far - 1024, ws_bytes=need, o=far) == INVALID  # the workspace runs into o
    # a short one needs none
    assert s3e.kv_attn_workspace(cache(), batch(max_kv=64), 4, s3e.TYPE_F32) == 0


def test_layout_of_reference_is_one_to_one():
    """The numpy layout the GPU tests compare with: every code and scale has bytes of its own, none left over."""
    import kv_ref

    for t in (kv_ref.Q4_0, kv_ref.Q8_0):
        for D in (32, 96):
            seen, scales = set(), set()
            for slot in range(32):
                for tensor in range(2):
                    for ch in range(D):
                        at, shift, sc = kv_ref.place(t, D, 32, 1, slot, 0, tensor, ch)
                        seen.add((at, shift))
                        scales.add(sc)
            assert len(seen) == 64 * D and len(scales) == 64 * D // 32
            used = {a for a, _ in seen} | scales | {s + 1 for s in scales}
            assert used == set(range(kv_ref.chunk_bytes(t, D)))
    x = np.array([[1.0, -1.0] + [0.5] * 30], np.float32)  # equal magnitudes: the first leads
    q, d = kv_ref.quantize(kv_ref.Q4_0, x)
    assert d.view(np.float16)[0, 0] == -0.125 and q[0, 0] == 0 and q[0, 1] == 15 and q[0, 2] == 4
