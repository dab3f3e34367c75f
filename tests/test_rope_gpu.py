"""Rotary positions against the formula in 64 bits."""
import numpy as np
import pytest
import torch

import kv8_ref as ref
from breccia_b200._lib import BrcError
from breccia_b200.qsa import Rope

pytestmark = pytest.mark.gpu

THETA = 500000.0
SCALINGS = {"none": {}, "linear": dict(factor=4.0), "ntk": dict(factor=8.0), "yarn": dict(factor=16.0, orig_ctx=8192),
            "bands": dict(factor=8.0, orig_ctx=8192)}
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def tolerance(x, want, m, dtype):
    """f32 arithmetic on the pair: cos and sin (times the factor, in 64 bits) rounded once, two products and a sum of three roundings
    of 2^-24 of the terms: within 8 * 2^-24 * (|x| + |y|) m; then the type's half step, and below its normal range half its
    least spacing."""
    fi = torch.finfo(dtype)
    pair = np.abs(x).max(-1, keepdims=True) * 2
    return 8 * 2.0 ** -24 * pair * m + (fi.eps / 2 * np.abs(want) if dtype != torch.float32 else 0) + fi.tiny * fi.eps


def check(got, x, want, m, dtype):
    got = got.double().cpu().numpy()
    assert (np.abs(got - want) <= tolerance(x, want, m, dtype)).all(), np.abs(got - want).max()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("scaling", list(SCALINGS))
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_scalings_layouts_types(cuda_device, layout, scaling, dtype):
    dt, n_rot, hd = DTYPES[dtype], 96, 128
    rope = Rope(n_rot, theta=THETA, layout=layout, scaling=scaling, **SCALINGS[scaling])
    g = torch.Generator(device="cuda").manual_seed(5)
    q = torch.randn(37, 5, hd, device="cuda", generator=g).to(dt)
    k = torch.randn(37, 2, hd, device="cuda", generator=g).to(dt)
    pos = np.concatenate([[0, 1, 2, 131071, 2 ** 20, 2 ** 31 - 1], np.arange(1000, 1031)]).astype(np.int32)
    freqs = ref.rope_freqs(n_rot, THETA, scaling, **SCALINGS[scaling])
    qo, ko = rope.apply(q, k, torch.from_numpy(pos).cuda())
    for x, y in ((q, qo), (k, ko)):
        xn = x.double().cpu().numpy()
        # a frequency in 64 bits is off by 2^-53 of itself: at position p that is p f 2^-52 of angle (f, and 2 pi, one rounding each)
        slack = 2.0 ** -51 * pos[:, None, None].astype(np.float64) * np.abs(xn).max() * rope.factor * 2
        want = ref.rotate(xn, pos, freqs, layout, rope.factor)
        err = np.abs(y.double().cpu().numpy() - want)
        assert (err <= tolerance(xn, want, rope.factor, dt) + slack).all(), err.max()


@pytest.mark.parametrize("tokens,heads,hd,n_rot", [(1, 1, 128, 2), (1, 16, 256, 256), (3, 7, 128, 90), (1001, 3, 80, 80), (2500, 2, 256, 16),
                                                   (5, 2, 64, 48), (700, 1, 33, 10)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_sizes(cuda_device, tokens, heads, hd, n_rot, layout):
    rope = Rope(n_rot, layout=layout)
    x = torch.randn(tokens, heads, hd, device="cuda", generator=torch.Generator(device="cuda").manual_seed(tokens)).half()
    pos = np.arange(tokens, dtype=np.int32) * 3
    y, none = rope.apply(x, None, torch.from_numpy(pos).cuda())
    assert none is None
    xn = x.double().cpu().numpy()
    check(y, xn, ref.rotate(xn, pos, ref.rope_freqs(n_rot, 10000.0), layout), 1.0, torch.float16)
    assert torch.equal(y[..., n_rot:], x[..., n_rot:])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("offset", [0, 1])
def test_columns_of_one_projection_in_place(cuda_device, layout, offset):
    """q and k as column blocks of a wider row, rotated where they lie; offset 1: rows that no 16-byte access fits."""
    n_q, n_kv, hd, tokens = 4, 2, 128, 19
    row = (n_q + 2 * n_kv) * hd + offset
    store = torch.randn(tokens * row + offset, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).bfloat16()
    before = store.clone()
    rope = Rope(64, layout=layout)

    def rows(t):
        m = t[offset:].view(tokens, row)
        return m[:, :n_q * hd].unflatten(1, (n_q, hd)), m[:, n_q * hd:(n_q + n_kv) * hd].unflatten(1, (n_kv, hd)), m[:, (n_q + n_kv) * hd:]

    q, k, rest = rows(store)
    pos = torch.arange(7, 7 + tokens, dtype=torch.int32, device="cuda")
    rope.apply(q, k, pos, q_out=q, k_out=k)
    q0, k0, rest0 = rows(before)
    qs, ks = rope.apply(q0.contiguous(), k0.contiguous(), pos)
    assert torch.equal(q, qs) and torch.equal(k, ks) and torch.equal(rest, rest0)


def test_offsets_past_32_bits(cuda_device):
    """More than 2^32 values, rotated in place: the last tokens as by themselves."""
    tokens = 2 ** 21 + 3
    x = torch.zeros(tokens, 16, 128, dtype=torch.float16, device="cuda")
    x[-5:] = torch.randn(5, 16, 128, device="cuda")
    x[0] = 1
    last, first = x[-5:].clone(), x[:1].clone()
    pos = torch.arange(tokens, dtype=torch.int32, device="cuda")
    rope = Rope(128, layout="interleaved")
    rope.apply(x, None, pos, q_out=x)
    assert torch.equal(x[-5:], rope.apply(last, None, pos[-5:].contiguous())[0]) and torch.equal(x[:1], first)
    assert x[1:-5].abs().max() == 0


def test_relative_positions(cuda_device):
    """The dot product of rotated q and k depends on the distance alone, at far positions too."""
    rope = Rope(128, theta=THETA, layout="interleaved")
    x = torch.randn(2, 1, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    dots = []
    for at in (0, 10 ** 6, 2 ** 31 - 200):
        y, _ = rope.apply(x, None, torch.tensor([at, at + 100], dtype=torch.int32, device="cuda"))
        dots.append(float((y[0].double() * y[1].double()).sum()))
    # 128 products of values off by 8 * 2^-24 * 2 max|x| each
    assert max(dots) - min(dots) <= 128 * 2 * 16 * 2.0 ** -24 * float(x.abs().max()) ** 2


def test_other_stream_and_graph(cuda_device):
    rope = Rope(64)
    x = torch.randn(9, 4, 128, device="cuda")
    pos = torch.arange(9, dtype=torch.int32, device="cuda")
    want, _ = rope.apply(x, None, pos)
    y = torch.zeros_like(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        rope.apply(x, None, pos, q_out=y)
    s.synchronize()
    assert torch.equal(y, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        rope.apply(x, None, pos, q_out=y)
    pos += 5
    g.replay()
    assert torch.equal(y, rope.apply(x, None, pos)[0])


def test_refusals(cuda_device):
    rope = Rope(64)
    x = torch.zeros(4, 2, 128, device="cuda")
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")
    for bad in (lambda: rope.apply(x.double(), None, pos), lambda: rope.apply(x[..., :32].contiguous(), None, pos),
                lambda: rope.apply(x, x[:3], pos), lambda: rope.apply(x, None, pos.long()), lambda: rope.apply(x, None, pos[:3]),
                lambda: rope.apply(x, None, pos.cpu()), lambda: rope.apply(x.transpose(1, 2), None, pos),
                lambda: rope.apply(x[:3], None, pos[:3], q_out=x[1:]), lambda: rope.apply(x, x.half(), pos),
                lambda: rope.apply(x.cpu(), None, pos)):
        with pytest.raises(BrcError):
            bad()
    assert rope.apply(x[:0], None, pos[:0])[0].shape == (0, 2, 128)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("hd,n_rot", [(128, 128), (256, 90), (80, 80)])   # rows of the wide kernel, of its odd pairing, of the other one
def test_negative_positions_turn_backwards(cuda_device, layout, hd, n_rot):
    rope = Rope(n_rot, theta=THETA, layout=layout, scaling="linear", factor=4.0)
    x = torch.randn(6, 3, hd, device="cuda", generator=torch.Generator(device="cuda").manual_seed(7))
    pos = np.array([-1, -7, -131072, -2 ** 31, 0, 9], np.int32)
    xn, freqs = x.double().cpu().numpy(), ref.rope_freqs(n_rot, THETA, "linear", 4.0)
    slack = 2.0 ** -51 * np.abs(pos[:, None, None].astype(np.float64)) * np.abs(xn).max() * 2   # as in test_scalings_layouts_types
    y, _ = rope.apply(x, None, torch.from_numpy(pos).cuda())
    want = ref.rotate(xn, pos, freqs, layout)
    assert (np.abs(y.double().cpu().numpy() - want) <= tolerance(xn, want, 1.0, torch.float32) + slack).all()
    # unsigned words are what they say: the same bits far forward
    y, _ = rope.apply(x, None, torch.from_numpy(pos.view(np.uint32)).cuda())
    far = pos.astype(np.int64) % 2 ** 32
    want = ref.rotate(xn, far, freqs, layout)
    slack = 2.0 ** -51 * far[:, None, None].astype(np.float64) * np.abs(xn).max() * 2
    assert (np.abs(y.double().cpu().numpy() - want) <= tolerance(xn, want, 1.0, torch.float32) + slack).all()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("hd,n_rot", [(256, 256), (256, 192), (256, 90), (256, 8), (64, 64), (64, 24), (128, 100)])
def test_every_row_kernel(cuda_device, layout, dtype, hd, n_rot):
    """Rows of one and of two chunks a lane, pairs by shuffle within a chunk, across chunks and through shared memory, beside untouched values."""
    rope = Rope(n_rot, layout=layout)
    g = torch.Generator(device="cuda").manual_seed(hd + n_rot)
    q, k = (torch.randn(37, h, hd, device="cuda", generator=g).to(DTYPES[dtype]) for h in (9, 2))
    pos = np.arange(37, dtype=np.int32) * 977
    out = rope.apply(q, k, torch.from_numpy(pos).cuda())
    for x, y in zip((q, k), out):
        xn = x.double().cpu().numpy()
        check(y, xn, ref.rotate(xn, pos, ref.rope_freqs(n_rot, 10000.0), layout), 1.0, DTYPES[dtype])
        assert torch.equal(y[..., n_rot:], x[..., n_rot:])
