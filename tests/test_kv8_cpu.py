"""8-bit pages and rotary positions without a GPU: the reference model itself, the frequencies, and the refusals that come before any
device is touched."""
import ctypes as C

import numpy as np
import pytest
import torch

import kv8_ref as ref
from breccia_b200 import _lib


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_reference_encoding(code):
    g = np.random.default_rng(1)
    x = np.concatenate([g.uniform(-1, 1, 4000) * ref.TOP[code], g.uniform(-1, 1, 4000) * 0.05, np.arange(-200, 200) / 512.0, [0.0, 1e9, -1e9]])
    y = ref.encode(x, code)
    if code == "e4m3":
        want = torch.from_numpy(np.clip(x, -448, 448)).to(torch.float32).to(torch.float8_e4m3fn).double().numpy()
        same = x.astype(np.float32) == x   # torch rounds from f32
        assert np.array_equal(y[same], want[same])
    assert np.all(np.abs(y - np.clip(x, -ref.TOP[code], ref.TOP[code])) <= ref.step_of(x, code) / 2)
    for amax in (1e-40, 0.0, 1.0, 127.0, 127.0001, 448.0, 448.1, 3e38, 2.0 ** -113 * 1.8):
        e = ref.exponent(amax, code)
        # the clamp: what needs more than 2^120 (int8 above 127 * 2^120) saturates
        assert (e == 120 or amax <= ref.TOP[code] * 2.0 ** e) and (e == -120 or amax > ref.TOP[code] * 2.0 ** (e - 1))


@pytest.mark.parametrize("scaling,more", [("none", {}), ("linear", dict(factor=4.0)), ("ntk", dict(factor=8.0)),
                                          ("yarn", dict(factor=16.0, orig_ctx=8192)), ("bands", dict(factor=8.0, orig_ctx=8192))])
@pytest.mark.parametrize("n_rot", [2, 64, 90, 256])
def test_frequencies(scaling, more, n_rot):
    from breccia_b200.qsa import Rope

    rope = Rope(n_rot, theta=500000.0, scaling=scaling, **more)
    want = ref.rope_freqs(n_rot, 500000.0, scaling, **more) / (2 * np.pi)
    got = rope.turns_host.astype(np.float64) * 2.0 ** -64
    # 0.64 fixed point: half of 2^-64; the reference: a few roundings of 2^-53
    assert np.all(np.abs(got - want) <= 2.0 ** -65 + 16 * 2.0 ** -53 * want)
    assert rope.factor == pytest.approx(0.1 * np.log(16.0) + 1 if scaling == "yarn" else 1.0, rel=2.0 ** -23)
    assert Rope(n_rot, scaling=scaling, mscale=1.25, **more).factor == 1.25


@pytest.mark.parametrize("bad", [dict(n_rot=3), dict(n_rot=0), dict(n_rot=258), dict(n_rot=64, theta=0.5), dict(n_rot=64, theta=float("nan")),
                                 dict(n_rot=64, scaling="linear", factor=0.5), dict(n_rot=64, scaling="yarn", factor=2.0),
                                 dict(n_rot=64, scaling="bands", factor=2.0, orig_ctx=8192, turns_low=4.0, turns_high=4.0),
                                 dict(n_rot=64, mscale=-1.0), dict(n_rot=64, layout="pairs"), dict(n_rot=64, scaling="log"),
                                 dict(n_rot=64, theta=1.0, scaling="yarn", factor=2.0, orig_ctx=8192)])
def test_frequency_refusals(bad):
    from breccia_b200.qsa import Rope

    with pytest.raises(_lib.BrcError):
        Rope(**bad)


def test_rope_apply_refusals():
    L = _lib.load()
    d = 0x1000

    def call(q=d, qo=d, nh=4, qs=0, qos=0, k=0, ko=0, nk=0, ks=0, kos=0, hd=128, dt=0, pos=d, n=3, turns=d, rot=64, lay=0):
        return L.brc_rope_apply(0, q, qo, nh, qs, qos, k, ko, nk, ks, kos, hd, dt, pos, n, turns, rot, lay, 1.0, None)

    for bad in (dict(dt=3), dict(lay=2), dict(hd=0), dict(rot=0), dict(rot=63), dict(rot=130), dict(q=0, qo=0), dict(qo=0), dict(nh=0),
                dict(qs=511), dict(qos=511), dict(pos=0), dict(turns=0), dict(q=d + 2, qo=d + 2), dict(qo=d + 16), dict(k=d, ko=d + 512, nk=1)):
        assert call(**bad) in (_lib.ERR_INVALID, _lib.ERR_UNSUPPORTED), bad
    assert call(n=0) == 0


def test_rope_outputs_that_touch_other_rows_are_refused():
    """Pointers are compared before any device is touched: with a NULL position pointer a call that passes that check fails at the next."""
    L = _lib.load()
    turns = (C.c_uint64 * 32)()

    def overlap(q, qo, k, ko, qs=0, qos=0, ks=0, kos=0, n=4, q_heads=4):   # heads of 64 in f32: 256 bytes each
        rc = L.brc_rope_apply(0, q, qo, q_heads, qs, qos, k, ko, 2 if k else 0, ks, kos, 64, 0, None, n, C.cast(turns, C.c_void_p), 64, 0, 1.0, None)
        assert rc == _lib.ERR_INVALID
        return b"overlap" in L.brc_last_error()

    a, b = 1 << 20, 2 << 20
    assert not overlap(a, a, b, b) and not overlap(a, a + 4096, b, b + 2048)
    assert overlap(a, a + 256, None, None) and overlap(a, a + 4092, None, None) and overlap(a, a, None, None, qs=512)
    assert not overlap(a, a, None, None, qs=512, n=1)
    wide = dict(qs=512, qos=512, ks=512, kos=512)                          # 2048 bytes a token: q 1024, k 512, the rest
    assert not overlap(a, a, a + 1024, a + 1024, **wide)                   # both in place, side by side
    assert not overlap(a, b, a + 1024, b + 1024, **wide)
    assert not overlap(a, a, a + 1024, a + 1536, **wide)                   # k to columns of its own
    assert overlap(a, a, a + 768, a + 1024, **wide)                        # k's rows are q's last head
    assert overlap(a, b, b + 512, b + 1536, **wide)                        # q's output ends inside k
    assert overlap(a, b, a + 1024, b + 2048 * 3 + 512, **wide)             # in the last row alone
    assert overlap(a, b, a + 1024, b + 1792, **wide)                       # k's output ends in q's next row
    assert overlap(a, b, b, b, ks=512, kos=512) and overlap(a, b, a + 1024, b, **wide)
    assert overlap(a, b + 1024, b, b, n=1) is False and overlap(a, b, b, b, n=1)


def test_rows_that_share_memory_are_refused():
    """A token broadcast over a batch has stride 0, which would be read as packed rows: past its end."""
    from breccia_b200.qsa import _token_rows

    wide = torch.zeros(4, 3 * 2 * 64)
    assert _token_rows(wide[:, 128:256].unflatten(1, (2, 64)), 2, 64, "x") == 384
    assert _token_rows(torch.zeros(1, 2, 64).expand(1, 2, 64), 2, 64, "x") == 128
    for bad in (torch.zeros(1, 2, 64).expand(4, 2, 64), torch.zeros(1, 128).expand(4, 128), torch.zeros(4, 1, 64).expand(4, 2, 64),
                torch.zeros(1024).as_strided((4, 2, 64), (64, 64, 1)), torch.zeros(1, 1, 64).expand(4, 1, 64)):
        with pytest.raises(_lib.BrcError):
            _token_rows(bad, bad.shape[1] if bad.dim() == 3 else 2, 64, "x")


def test_pool_refusals():
    L = _lib.load()
    h = C.c_void_p()
    for args, rc in (((0, 1, 2, 256, 16, 8, 3), _lib.ERR_INVALID), ((0, 1, 2, 96, 16, 8, 1), _lib.ERR_UNSUPPORTED),
                     ((0, 1, 2, 256, 32, 8, 1), _lib.ERR_UNSUPPORTED), ((0, 0, 2, 256, 16, 8, 2), _lib.ERR_INVALID)):
        assert L.brc_pool_create_kv8(*args, C.byref(h)) == rc and not h.value
    if not torch.cuda.is_available():
        assert L.brc_pool_create_kv8(0, 1, 2, 256, 16, 8, 1, C.byref(h)) == _lib.ERR_CUDA
    from breccia_b200.qsa import KvPool

    for bad in (dict(kv8="fp8"), dict(kv8="int8", v_q8=True), dict(kv8="int8", bookkeeping_only=True)):
        with pytest.raises(_lib.BrcError):
            KvPool(0, 1, 2, 256, 8, **bad)
    book = KvPool(0, 1, 2, 256, 8, bookkeeping_only=True)
    code, b = C.c_int32(7), C.c_uint64()
    assert L.brc_pool_kv8_code(book.handle, C.byref(code)) == 0 and code.value == 0
    d = C.c_void_p(0x1000)
    assert L.brc_kv8_append(book.handle, 0, d, 4, d, 1, 1, None, 1, 1, d, 0, d, 0, 0, None, 0, 0, 1.0, None) == _lib.ERR_CUDA
    assert L.brc_kv8_read(book.handle, 0, d, 4, d, 1, 1, None, 1, 1, d, d, 0, None) == _lib.ERR_CUDA
    assert L.brc_kv8_attn(book.handle, 0, d, 1, 16, None, 0, d, 4, d, None, 1, 1, 16, 1.0, d, 1, d, 1 << 30, None) == _lib.ERR_CUDA
    assert L.brc_kv8_attn_workspace_bytes(book.handle, 1, 16, 1, C.byref(b)) == _lib.ERR_UNSUPPORTED
    for null in (lambda: L.brc_kv8_append(None, 0, d, 4, d, 1, 1, None, 1, 1, d, 0, d, 0, 0, None, 0, 0, 1.0, None),
                 lambda: L.brc_kv8_attn_workspace_bytes(None, 1, 16, 1, C.byref(b)), lambda: L.brc_pool_kv8_code(None, C.byref(code))):
        assert null() == _lib.ERR_INVALID


def test_ragged_attention_refusals():
    L = _lib.load()
    from breccia_b200.qsa import KvPool

    book, d = KvPool(0, 1, 2, 256, 8, bookkeeping_only=True), C.c_void_p(0x1000)

    def call(pool=book.handle, total=3, cu=d):
        return L.brc_kv8_attn_ragged(pool, 0, d, 1, total, 16, None, 0, d, 4, d, cu, 1, 3, 16, 1.0, d, 1, d, 1 << 30, None)

    assert call() == _lib.ERR_CUDA and b"brc_kv8_attn_ragged" in L.brc_last_error()
    assert call(cu=None) == _lib.ERR_INVALID and b"NULL prefix" in L.brc_last_error()
    assert call(pool=None) == _lib.ERR_INVALID


def test_rope_layouts_with_signed_positions():
    L, d = _lib.load(), 0x1000
    for layout, ok in ((0, True), (1, True), (256, True), (257, True), (2, False), (258, False), (512, False), (-1, False)):
        rc = L.brc_rope_apply(0, d, d, 1, 0, 0, None, None, 0, 0, 0, 64, 0, d, 0, d, 64, layout, 1.0, None)
        assert (rc == 0) == ok and (ok or rc == _lib.ERR_INVALID), layout


def test_attention_arguments_that_describe_no_memory():
    """Strides and views that the library, given an address and a size, would read past: refused in front of it (which would answer
    ERR_CUDA for this pool without a device)."""
    from breccia_b200.qsa import KvPool, kv8_attend

    pool = KvPool(0, 1, 2, 128, 8, bookkeeping_only=True)
    pool.device = -1   # where CPU tensors lie
    q, t, n, ws = torch.ones(2, 4, 128), torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32), torch.zeros(1 << 20, dtype=torch.uint8)
    gate = torch.ones(2, 4, 128)
    for bad in (dict(gate=gate, gate_head_stride=-128), dict(gate=gate, gate_head_stride=0), dict(gate=gate, gate_head_stride=64),
                dict(gate=gate[:1], gate_head_stride=128), dict(gate=gate[:0], gate_head_stride=128), dict(ws=ws[:1].expand(1 << 20)), dict(ws=ws[::2])):
        with pytest.raises(_lib.BrcError) as e:
            kv8_attend(pool, 0, q, t, n, 16, bad.pop("ws", ws), **bad)
        assert e.value.code == _lib.ERR_INVALID, bad


def test_rope_refuses_more_tokens_than_a_call_counts():
    """2^32 + 1 rows are one row to a 32-bit count; meta tensors have the shape without the memory."""
    from breccia_b200.qsa import Rope

    rope = Rope(2)
    rope.device = -1   # where meta tensors lie
    for n in (2 ** 32, 2 ** 32 + 1):
        x, pos = torch.empty(n, 1, 2, dtype=torch.float16, device="meta"), torch.empty(n, dtype=torch.int32, device="meta")
        with pytest.raises(_lib.BrcError, match="tokens"):
            rope.apply(x, None, pos, q_out=x)
