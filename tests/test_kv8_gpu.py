"""8-bit pages: the quantising write (bit-exact), the read-back and attention against plain 64-bit numpy (kv8_ref.py)."""
import math

import numpy as np
import pytest
import torch

import kv8_ref as ref
from breccia_b200 import _lib, synth
from breccia_b200._lib import BrcError
from breccia_b200.qsa import DecodeBatch, KvPool, Rope, kv8_append, kv8_attend, kv8_read, kv8_workspace

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
NAN, INF = float("nan"), float("inf")


def dev(a, dtype=np.int32):
    return torch.from_numpy(np.ascontiguousarray(a, dtype)).cuda()


def scattered(seed, needs, spare=3):
    """Tables for sequences of needs[s] cells in a shuffled pool."""
    pages = [-(-n // 16) for n in needs]
    ids = synth.permutation(seed, sum(pages) + spare)
    t = np.full((len(needs), max(max(pages), 1)), 0, np.int32)
    at = 0
    for s, n in enumerate(pages):
        t[s, :n] = ids[at:at + n]
        at += n
    return t, sum(pages) + spare


def random_rows(g, total, n_kv, hd, dtype):
    """Rows whose size drifts, so that scales grow inside a page."""
    x = torch.randn(total, n_kv, hd, device="cuda", generator=g) * torch.exp(1.5 * torch.randn(total, n_kv, 1, device="cuda", generator=g))
    return x.to(DTYPES[dtype])


def assert_pool_is(pool, cache, tables, lens, layer=0):
    """Codes (as the values they stand for in units of the scale) and scales of every written cell, bit for bit."""
    for side in (0, 1):
        codes, scales = (x.float().cpu().numpy() for x in pool.kv8_view(side, layer))
        for s, n in enumerate(lens):
            for j in range(-(-n // 16)):
                i, live = tables[s][j], min(16, n - 16 * j)
                for h in range(pool.n_kv_head):
                    page = cache.p[i][h][side]
                    assert scales[i, h] == 2.0 ** page.e, (s, j, h, side)
                    assert np.array_equal(codes[i, h, :live], page.c[:live]), (s, j, h, side)


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n_kv,hd", [(2, 256), (3, 128)])
def test_append_in_pieces_is_bit_exact(cuda_device, code, dtype, n_kv, hd):
    """Ragged pieces of 0, 1, 15, 16, 17 and 40 tokens, page by page, through scattered tables; then back as values."""
    steps = [[1, 17, 0, 40], [1, 15, 16, 1], [14, 0, 1, 16], [1, 1, 1, 0], [40, 3, 17, 33]]
    lens = np.sum(steps, 0)
    tables, n_pages = scattered(3, lens + 5)
    pool = KvPool(0, 2, n_kv, hd, n_pages, kv8=code)
    pool.poison_nan()
    cache = ref.Cache(n_pages, n_kv, hd, code)
    t, g = dev(tables), torch.Generator(device="cuda").manual_seed(4)
    at = np.zeros(4, np.int64)
    for counts in steps:
        total = sum(counts)
        k, v = random_rows(g, total, n_kv, hd, dtype), random_rows(g, total, n_kv, hd, dtype)
        cu = np.concatenate([[0], np.cumsum(counts)])
        kv8_append(pool, 1, k, v, t, dev(at), int((at + counts).max()), cu_tokens=dev(cu))
        kn, vn = k.double().cpu().numpy(), v.double().cpu().numpy()
        for s in range(4):
            cache.append(tables[s], int(at[s]), kn[cu[s]:cu[s + 1]], vn[cu[s]:cu[s + 1]])
        at += counts
    pool.check()
    assert_pool_is(pool, cache, tables, lens, layer=1)
    cu = np.concatenate([[0], np.cumsum(lens)])
    for out, dt in DTYPES.items():
        got = kv8_read(pool, 1, t, dev(np.zeros(4)), int(lens.max()), cu_tokens=dev(cu), total_tokens=int(cu[-1]), dtype=dt)
        for side in (0, 1):
            want = torch.from_numpy(np.concatenate([cache.values(tables[s], int(lens[s]), side) for s in range(4)]))
            assert torch.equal(got[side].cpu(), want.to(dt)), (out, side)   # one rounding of an exact f32 number
    pool.check()
    pool.release()


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_read_back_windows_leave_the_rest(cuda_device, code):
    pool = KvPool(0, 1, 2, 128, 12, kv8=code)
    g = torch.Generator(device="cuda").manual_seed(1)
    t = dev(np.arange(10)[None])
    k, v = random_rows(g, 150, 2, 128, "f32"), random_rows(g, 150, 2, 128, "f32")
    kv8_append(pool, 0, k, v, t, dev([0]), 150, tokens_per_seq=150)
    whole = kv8_read(pool, 0, t, dev([0]), 150, tokens_per_seq=150, dtype=torch.float32)
    for p, n in ((0, 1), (15, 1), (15, 2), (16, 16), (17, 31), (1, 149), (149, 1)):
        part = kv8_read(pool, 0, t, dev([p]), p + n, tokens_per_seq=n, dtype=torch.float32)
        assert all(torch.equal(a, b[p:p + n]) for a, b in zip(part, whole)), (p, n)
    pool.check()
    pool.release()


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_infinities_nan_zeros_and_the_ends_of_the_range(cuda_device, code):
    pool = KvPool(0, 1, 1, 128, 8, kv8=code)
    cache = ref.Cache(8, 1, 128, code)
    rows = torch.zeros(6 * 16, 1, 128)
    rows[0, 0, :4] = torch.tensor([INF, -INF, NAN, 1.0])
    rows[16] = 1e-38                                   # far below the least scale
    rows[17, 0, 0] = 2.0 ** -118
    rows[32, 0, :2] = torch.tensor([3.3e38, -1.0])     # above what int8's greatest scale reaches
    rows[48, 0, :] = torch.linspace(-448, 448, 128)
    rows[64, 0, :] = torch.arange(128) / 128.0 * 127   # ties
    rows[80:] = INF                                    # nothing finite
    k = rows.cuda()
    kv8_append(pool, 0, k, -k, dev(np.arange(6)[None]), dev([0]), 96, tokens_per_seq=96)
    with pytest.raises(BrcError, match="infinity or NaN"):
        pool.check()
    cache.append(np.arange(6), 0, rows.double().numpy(), -rows.double().numpy())
    assert_pool_is(pool, cache, [np.arange(6)], [96])
    pool.check()
    pool.release()


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_rolling_back_and_the_page_of_another_sequence(cuda_device, code):
    """An append at a smaller pos0 keeps what lies in front of it; a page taken over from another sequence starts afresh."""
    pool = KvPool(0, 1, 2, 128, 4, kv8=code)
    cache = ref.Cache(4, 2, 128, code)
    g = torch.Generator(device="cuda").manual_seed(8)
    t = dev([[2, 0]])
    for p, n, size in ((0, 21, 1.0), (18, 2, 30.0), (18, 1, 0.01), (7, 4, 1e4), (0, 3, 1e-3)):
        k, v = (random_rows(g, n, 2, 128, "f32") * size for _ in range(2))
        kv8_append(pool, 0, k, v, t, dev([p]), p + n, tokens_per_seq=n)
        cache.append([2, 0], p, k.double().cpu().numpy(), v.double().cpu().numpy())
        assert_pool_is(pool, cache, [[2, 0]], [min(p + n, 16) if p < 16 else p + n])
    pool.check()
    pool.release()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("n_rot,offset", [(128, 0), (64, 0), (90, 0), (64, 1)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_append_rotates_keys(cuda_device, layout, n_rot, offset, dtype):
    """K and V as column blocks of a wider row (offset 1: unaligned); K rotated by its cell's position."""
    n_kv, hd, code = 2, 128, "int8"
    counts, pos0 = [33, 1, 20], [1005, 131000, 5]
    tables, n_pages = scattered(5, [p % 16 + n + 16 for p, n in zip(pos0, counts)])
    wide = np.zeros((3, 131072 // 16 + 4), np.int32)
    for s, p in enumerate(pos0):
        wide[s, p // 16:p // 16 + tables.shape[1]] = tables[s][:wide.shape[1] - p // 16]
    g = torch.Generator(device="cuda").manual_seed(2)
    total, row = sum(counts), 2 * n_kv * hd + offset
    store = torch.randn(total * row + offset, device="cuda", generator=g).to(DTYPES[dtype])
    m = store[offset:].view(total, row)
    k, v = m[:, :n_kv * hd], m[:, n_kv * hd:2 * n_kv * hd]
    pool = KvPool(0, 1, n_kv, hd, n_pages, kv8=code)
    rope = Rope(n_rot, theta=500000.0, layout=layout, scaling="yarn", factor=16.0, orig_ctx=8192)
    cu = np.concatenate([[0], np.cumsum(counts)])
    kv8_append(pool, 0, k, v, dev(wide), dev(pos0), 131072, cu_tokens=dev(cu), rope=rope)
    got_k, got_v = kv8_read(pool, 0, dev(wide), dev(pos0), 131072, cu_tokens=dev(cu), total_tokens=total, dtype=torch.float32)
    pool.check()
    freqs = ref.rope_freqs(n_rot, 500000.0, "yarn", 16.0, 8192)
    pos = np.concatenate([np.arange(p, p + n) for p, n in zip(pos0, counts)])
    xk = ref.rotate(k.double().cpu().numpy().reshape(total, n_kv, hd), pos, freqs, layout, rope.factor)
    xv = v.double().cpu().numpy().reshape(total, n_kv, hd)
    # int8: half a step of the page's scale; K also the rotation's f32 error (test_rope_gpu.tolerance: 8 * 2^-24 * 2 max|x| m),
    # which may move a value over the border to the next code: twice that, on top of the half step
    fuzz = 2 * 8 * 2.0 ** -24 * 2 * np.abs(m.double().cpu().numpy()).max() * rope.factor
    for x, got, f in ((xk, got_k, fuzz), (xv, got_v, 0.0)):
        got = got.double().cpu().numpy()
        for s in range(3):
            for a in range(cu[s], cu[s + 1]):
                p = pos[a]
                page = [b for b in range(cu[s], cu[s + 1]) if pos[b] // 16 == p // 16]
                for h in range(n_kv):
                    amax = np.abs(x[page, h]).max()
                    step = 2.0 ** ref.exponent(amax * (1 + f / amax), "int8")
                    assert np.abs(got[a, h] - x[a, h]).max() <= step / 2 + f, (s, a, h)
    pool.release()


def test_bad_pages_and_positions_are_skipped_and_reported(cuda_device):
    pool = KvPool(0, 1, 2, 128, 4, kv8="e4m3")
    k = torch.ones(40, 2, 128, device="cuda")
    kv8_append(pool, 0, k, k, dev([[0, 9, 1]]), dev([0]), 40, tokens_per_seq=40)
    with pytest.raises(BrcError, match="page id"):
        pool.check()
    kv8_append(pool, 0, k, k, dev([[0, 2, 1]]), dev([0]), 20, tokens_per_seq=40)     # cells 20 .. are past the caller's bound
    with pytest.raises(BrcError, match="position past bound"):
        pool.check()
    got, _ = kv8_read(pool, 0, dev([[0, 2, 1]]), dev([0]), 20, tokens_per_seq=20, dtype=torch.float32)
    assert torch.equal(got, k[:20])
    assert pool.kv8_view(0, 0)[0].float()[2, :, 4:].abs().max() == 0
    out = torch.full((1, 2, 40, 2, 128), 7.0, device="cuda")
    t, zero = dev([[9, 2, 1]]), dev([0])
    _lib.call("brc_kv8_read", pool.handle, 0, t.data_ptr(), 3, zero.data_ptr(), 1, 40, None, 40, 40, out[0, 0].data_ptr(),
              out[0, 1].data_ptr(), 0, torch.cuda.current_stream().cuda_stream)
    with pytest.raises(BrcError, match="page id"):
        pool.check()
    assert (out[0, 0, :16] == 7).all()
    # attention: the cells of a page out of range count as not there
    q = torch.randn(1, 2, 128, device="cuda")
    ws = kv8_workspace(pool, 1, 2)
    got = kv8_attend(pool, 0, q, dev([[0, 9]]), dev([20]), 32, ws)
    with pytest.raises(BrcError, match="page id"):
        pool.check()
    assert torch.equal(got, kv8_attend(pool, 0, q, dev([[0, 2]]), dev([16]), 32, ws))
    # a length past the bound is cut off there
    kv8_attend(pool, 0, q, dev([[0, 2]]), dev([21]), 20, ws)
    with pytest.raises(BrcError, match="position past bound"):
        pool.check()
    pool.release()


def test_refusals(cuda_device):
    pool = KvPool(0, 1, 2, 128, 4, kv8="int8")
    plain = KvPool(0, 1, 2, 128, 4)
    k, t, p = torch.ones(4, 2, 128, device="cuda"), dev([[0, 1]]), dev([0])
    q, lens, ws = torch.ones(1, 4, 128, device="cuda"), dev([4]), kv8_workspace(pool, 1, 4)
    for bad in (lambda: kv8_append(pool, 1, k, k, t, p, 4, 4), lambda: kv8_append(pool, 0, k, k, t, p, 33, 4),
                lambda: kv8_append(pool, 0, k, k, t, p, 4, 3), lambda: kv8_append(pool, 0, k.double(), k.double(), t, p, 4, 4),
                lambda: kv8_append(pool, 0, k, k[:3], t, p, 4, 4), lambda: kv8_append(pool, 0, k[:, :1], k[:, :1], t, p, 4, 4),
                lambda: kv8_append(pool, 0, k, k, t.long(), p, 4, 4), lambda: kv8_append(plain, 0, k, k, t, p, 4, 4),
                lambda: kv8_append(pool, 0, k.transpose(1, 2).contiguous(), k, t, p, 4, 4),
                lambda: kv8_append(pool, 0, k, k, t, p, 4, 4, rope=Rope(256)), lambda: kv8_append(pool, 0, k.cpu(), k.cpu(), t, p, 4, 4),
                lambda: kv8_read(pool, 0, t, p, 33, 4), lambda: kv8_read(plain, 0, t, p, 4, 4), lambda: kv8_read(pool, 0, t, p, 4, 4, dtype=torch.int8),
                lambda: kv8_read(pool, 0, t, p, 4, cu_tokens=dev([0, 4])),
                lambda: kv8_attend(pool, 1, q, t, lens, 4, ws), lambda: kv8_attend(pool, 0, q[:, :3].contiguous(), t, lens, 4, ws),
                lambda: kv8_attend(pool, 0, q, t, lens, 33, ws), lambda: kv8_attend(pool, 0, q, t, lens, 4, ws[:-16]),
                lambda: kv8_attend(pool, 0, q, t, lens, 4, ws, max_q=2), lambda: kv8_attend(plain, 0, q, t, lens, 4, ws),
                lambda: kv8_attend(pool, 0, q.half(), t, lens, 4, ws, out=torch.ones(1, 4, 128)), lambda: kv8_attend(pool, 0, q, t, lens.long(), 4, ws),
                lambda: kv8_attend(pool, 0, q, t, lens, 4, ws, gate=q, gate_head_stride=64), lambda: kv8_workspace(plain, 1, 4),
                lambda: kv8_attend(pool, 0, torch.ones(1, 4, 129, device="cuda").view(-1)[1:513].view(1, 4, 128), t, lens, 4, ws),
                lambda: plain.kv8_view(0, 0), lambda: pool.kv8_view(2, 0), lambda: pool.gather(0, t[0], 4)):
        with pytest.raises(BrcError):
            bad()
    L, d = _lib.load(), q.data_ptr()
    for rc in (L.brc_paged_prefill_attn(pool.handle, 0, d, 0, 4, None, 0, t.data_ptr(), 2, p.data_ptr(), 1, 1, 4, 1.0, d, None),
               L.brc_paged_sparse_attn(pool.handle, 0, d, 0, 4, None, 0, t.data_ptr(), 2, p.data_ptr(), 1, 1, t.data_ptr(), 1, p.data_ptr(), 4, 1.0, d, None),
               L.brc_decode_partial(pool.handle, 0, d, 0, 4, t.data_ptr(), 2, lens.data_ptr(), 1, 4, 1.0, d, ws.data_ptr(), ws.numel(), None),
               L.brc_paged_decode_attn_static(pool.handle, 0, d, 0, 4, None, 0, t.data_ptr(), 2, lens.data_ptr(), 1, 4, 1.0, d, None),
               L.brc_state_dump(pool.handle, 0, np.zeros(2, np.uint32).ctypes.data_as(_lib._u32p), 2, 4, 0, b"/tmp", None),
               L.brc_decode_step(pool.handle, 0, 1, t.data_ptr(), 2, lens.data_ptr(), p.data_ptr(), 1, 5, d, 0, 0, 4, d, d, 0, 0, None, 0, 0, 1.0, d, 0, ws.data_ptr(), ws.numel(), None)):
        assert rc == _lib.ERR_UNSUPPORTED
        assert b"8-bit" in L.brc_last_error()
    assert kv8_read(pool, 0, t, p, 0, 0)[0].shape == (0, 2, 128)
    kv8_append(pool, 0, k[:0], k[:0], t, p, 0, 0)
    pool.check()
    pool.release()
    plain.release()


# ------------------------------------------------------------------------------------------------- attention
def fill(pool, seed, layer=0):
    """Random pages straight into the pool: scales differ from page to page, head to head and side to side."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for side in (0, 1):
        codes, scales = pool.kv8_view(side, layer)
        x = torch.randn(codes.shape, device="cuda", generator=g) * (40 if pool.kv8 == "int8" else 100)
        codes.copy_(x.round().clamp(-127, 127).to(torch.int8) if pool.kv8 == "int8" else x.clamp(-448, 448).to(torch.float8_e4m3fn))
        scales.copy_(torch.exp2(torch.randint(-9, -4, scales.shape, device="cuda", generator=g).float()))
        out.append((codes.double() * scales.double()[..., None, None]).cpu().numpy())
    return out


def cells(values, table, n):
    if n == 0:
        return np.zeros((0,) + values.shape[1:2] + values.shape[3:])
    return np.concatenate([values[i].transpose(1, 0, 2) for i in table[: -(-n // 16)]])[:n]


def run_and_compare(pool, values, tables, lens, n_q, n_head, q_dt, out_dt, ragged, gate=False, seed=9, scale=None, table_dev=None, q_scale=1.5):
    hd, n_seqs = pool.head_dim, len(lens)
    g = torch.Generator(device="cuda").manual_seed(seed)
    cu = np.concatenate([[0], np.cumsum(n_q)])
    q = (torch.randn(int(cu[-1]), n_head, hd, device="cuda", generator=g) * q_scale).to(DTYPES[q_dt])
    gates = torch.randn(int(cu[-1]), n_head, 2 * hd, device="cuda", generator=g) if gate else None
    ws = kv8_workspace(pool, n_seqs, n_head, max(n_q))
    scale = 1 / math.sqrt(hd) if scale is None else scale
    got = kv8_attend(pool, 0, q, dev(tables) if table_dev is None else table_dev, dev(lens), int(max(lens)), ws, max_q=max(n_q), cu_q=dev(cu) if ragged else None,
                     scale=scale, out_dtype=DTYPES[out_dt], gate=gates, gate_head_stride=2 * hd if gate else 0)
    pool.check()
    assert got.dtype == DTYPES[out_dt]
    got, qn = got.double().cpu().numpy(), q.double().cpu().numpy()
    fi = torch.finfo(DTYPES[out_dt])
    worst = 0.0
    for s in range(n_seqs):
        k, v = (cells(x, tables[s], int(lens[s])) for x in values)
        for i in range(n_q[s]):
            row = cu[s] + i
            want, mag, dot = ref.attention(qn[row], k, v, int(lens[s]) - (n_q[s] - 1 - i), scale)
            if gate:
                sg = 1 / (1 + np.exp(-gates[row, :, :hd].double().cpu().numpy()))
                want, mag = want * sg, mag * sg
            # weights: the probabilities' binary16 rounding (2^-11; two parts: 2^-22) and the exponent's error - a dot product of
            # hd exact products accumulated in f32 over hd / 16 steps, each within 2^-22 of the sum of magnitudes, twice (score and
            # maximum), and exp2's own 2^-21; the sums over cells, a step of 2^-22 each 16 cells; numerator and denominator alike
            half = 2.0 ** -11 if q_dt != "f32" and out_dt != "f32" else 2.0 ** -21
            exponent = 2 * (hd / 16 + 4) * 2.0 ** -22 * dot[:, None] + 4 * 2.0 ** -21
            tol = mag * (half + 2 * exponent + 2 * (lens[s] / 16 + 32) * 2.0 ** -22) + (fi.eps / 2 * np.abs(want) if out_dt != "f32" else 0) + fi.tiny * fi.eps
            if gate:
                tol = tol + mag * 2.0 ** -20    # the sigmoid in f32
            err = np.abs(got[row] - want)
            assert (err <= tol).all(), (s, i, float((err - tol).max()), float(err.max()))
            worst = max(worst, float((err / (tol + 1e-300)).max()))
    return worst


LENS = [1, 0, 15, 16, 17, 300, 33, 1000]


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("q_dt,out_dt", [("f16", "f16"), ("bf16", "bf16"), ("f32", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("n_head,n_kv,hd", [(16, 2, 256), (5, 1, 256), (32, 8, 128), (7, 7, 128)])
def test_one_token_each(cuda_device, code, q_dt, out_dt, n_head, n_kv, hd):
    tables, n_pages = scattered(2, LENS)
    pool = KvPool(0, 1, n_kv, hd, n_pages, kv8=code)
    values = fill(pool, 3)
    run_and_compare(pool, values, tables, LENS, [1] * len(LENS), n_head, q_dt, out_dt, False)
    pool.release()


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("dt", ["f16", "f32"])
@pytest.mark.parametrize("n_head,n_kv,hd,n_q", [(16, 2, 256, [2] * 8), (8, 2, 256, [4, 1, 0, 3, 2, 4, 4, 4]), (32, 8, 128, [8, 0, 8, 8, 1, 5, 8, 8]),
                                                (24, 2, 256, [3, 1, 2, 3, 3, 3, 3, 3]), (40, 2, 128, [1, 1, 2, 2, 2, 2, 2, 2]), (3, 3, 128, [17] * 8)])
def test_several_tokens_gate_and_empty_rows(cuda_device, code, dt, n_head, n_kv, hd, n_q):
    """Ragged drafts, several passes of 32 rows, rows in front of the first cell (which see nothing), a gate."""
    tables, n_pages = scattered(2, LENS)
    pool = KvPool(0, 1, n_kv, hd, n_pages, kv8=code)
    values = fill(pool, 4)
    run_and_compare(pool, values, tables, LENS, n_q, n_head, dt, dt, len(set(n_q)) > 1, gate=True)
    pool.release()


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_long_sequences_split_over_every_sm(cuda_device, code):
    lens = [20011, 5, 9000]
    tables, n_pages = scattered(6, lens)
    pool = KvPool(0, 1, 2, 128, n_pages, kv8=code)
    values = fill(pool, 5)
    for dt in ("f16", "f32"):
        run_and_compare(pool, values, tables, lens, [1, 2, 3], 16, dt, dt, True)
    pool.release()


def test_nothing_to_attend_to(cuda_device):
    """Every sequence empty: zeros, whatever the workspace and the output held; no sequences, no tokens: nothing written."""
    pool = KvPool(0, 1, 2, 128, 4, kv8="int8")
    t, q = dev(np.zeros((5, 2))), torch.randn(10, 8, 128, device="cuda").half()
    ws, out = kv8_workspace(pool, 5, 8, 2), torch.full((10, 8, 128), 7.0, device="cuda").half()
    ws.fill_(255)
    for bound in (0, 32):
        out.fill_(7)
        kv8_attend(pool, 0, q, t, dev([0] * 5), bound, ws, max_q=2, out=out)
        pool.check()
        assert (out == 0).all()
    out.fill_(7)
    kv8_attend(pool, 0, q, t, dev([3] * 5), 32, ws, max_q=2, cu_q=dev([0, 0, 2, 2, 2, 2]), out=out)   # four sequences without tokens, rows behind the last one
    pool.check()
    assert (out[:2] == 0).all() and (out[2:] == 7).all()   # (zeros: a zeroed pool)
    assert kv8_attend(pool, 0, q[:0], t[:0], dev([]), 32, ws).shape == (0, 8, 128)
    pool.release()


def test_a_prefix_that_does_not_begin_at_zero(cuda_device):
    """Tokens in front of cu_tokens[0] belong to nobody; those behind the last entry neither."""
    pool = KvPool(0, 1, 1, 128, 8, kv8="e4m3")
    k = torch.randn(60, 1, 128, device="cuda")
    for first, n in ((3, 5), (40, 17), (16, 16)):
        pool.zero()
        kv8_append(pool, 0, k, k, dev([[4, 2]]), dev([1]), 32, cu_tokens=dev([first, first + n]))
        pool.check()
        got, _ = kv8_read(pool, 0, dev([[4, 2]]), dev([1]), 32, tokens_per_seq=n, dtype=torch.float32)
        # e4m3: half a step, 2^-4 of the value, below the least normal code 2^-10 of the scale (at most 2 max / 448)
        assert ((got - k[first:first + n]).abs() <= 2.0 ** -4 * k[first:first + n].abs() + 2.0 ** -10 * 2 * k.abs().max() / 448).all()
        codes = pool.kv8_view(0, 0)[0].float()
        assert codes[[0, 1, 3, 5, 6, 7]].abs().max() == 0 and codes[4, :, 0].abs().max() == 0
    pool.release()


def test_raw_pages_through_the_host(cuda_device):
    """read / write move whole half pages, codes and scales."""
    pool = KvPool(0, 1, 2, 128, 3, kv8="int8")
    fill(pool, 3)
    raw = pool.read(1, 0)
    assert raw.shape == (3, pool.half_page_bytes) and pool.half_page_bytes % 128 == 0
    codes, scales = (x.cpu().numpy() for x in pool.kv8_view(1, 0))
    assert np.array_equal(raw[:, :2 * 16 * 128].view(np.int8).reshape(3, 2, 16, 128), codes)
    assert np.array_equal(raw[:, 2 * 16 * 128:2 * 16 * 128 + 8].copy().view(np.float32), scales)
    pool.zero()
    pool.write(1, 0, raw)
    assert np.array_equal(pool.read(1, 0), raw) and pool.bytes() == 2 * 3 * pool.half_page_bytes
    pool.release()


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_offsets_past_32_bits(cuda_device, code):
    """A layer of more than 2^32 bytes: the same tokens in its first and its last pages, in the second of two layers."""
    n_pages = 300_000
    pool = KvPool(0, 2, 4, 256, n_pages, kv8=code)
    assert n_pages * pool.half_page_bytes > 2 ** 32
    t = dev([[3, 1, 2], [n_pages - 1, n_pages - 3, n_pages - 2]])
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (random_rows(g, 40, 4, 256, "f16").repeat(2, 1, 1) for _ in range(2))
    kv8_append(pool, 1, k, v, t, dev([0, 0]), 40, tokens_per_seq=40)
    got = kv8_read(pool, 1, t, dev([0, 0]), 40, tokens_per_seq=40, dtype=torch.float32)
    assert all(torch.equal(x[:40], x[40:]) and x.abs().max() > 0 for x in got)
    q = torch.randn(1, 8, 256, device="cuda").repeat(2, 1, 1)
    out = kv8_attend(pool, 1, q, t, dev([40, 40]), 48, kv8_workspace(pool, 2, 8))
    want, mag, dot = ref.attention(q[0].double().cpu().numpy(), *(x[:40].double().cpu().numpy() for x in got), 40, 1 / 16)
    # As in the serving run; and random rows this unlike in size leave columns whose heaviest cells have code 0, where what counts lies below
    # the least weight.  A weight is 2^(s + e_v - M + 7) in binary16, whose half spacing at zero is 2^-25, and the references lie at or
    # under the true maxima (so the denominator is at least 1): a cell loses at most 2^-32 of a code times 2^M, 2^M at most the largest
    # scale, and the largest code times that scale at most twice the largest value: 2^-31 max|v| a cell.
    floor = 40 * 2.0 ** -31 * float(got[1].abs().max())
    for row in out.double().cpu().numpy():   # (the two sequences are cut at different pages, so their f32 sums run in different orders)
        assert (np.abs(row - want) <= mag * 2.0 ** -17 * (1 + dot[:, None]) + floor).all()
    pool.check()
    pool.release()


def test_many_short_sequences(cuda_device):
    """More sequences than threads in the schedule's scan, most of them a page or none, sharing pages."""
    g = np.random.default_rng(0)
    lens = g.choice([0, 1, 5, 16, 31, 70], 1500)
    tables = g.integers(0, 40, (1500, 5)).astype(np.int32)
    pool = KvPool(0, 1, 2, 128, 40, kv8="int8")
    values = fill(pool, 6)
    run_and_compare(pool, values, tables, lens, [1] * 1500, 4, "f16", "f16", False)
    pool.release()


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_what_no_row_sees_may_hold_anything(cuda_device, code):
    """Cells behind the length, in its last page and in the pages behind it, are NaN, codes and scales."""
    lens = [1, 16, 37]
    tables, n_pages = scattered(2, [64, 64, 64])
    pool = KvPool(0, 1, 2, 128, n_pages, kv8=code)
    pool.poison_nan()
    g = torch.Generator(device="cuda").manual_seed(1)
    cu = np.concatenate([[0], np.cumsum(lens)])
    k, v = random_rows(g, 54, 2, 128, "f16"), random_rows(g, 54, 2, 128, "f16")
    t = dev(tables)
    kv8_append(pool, 0, k, v, t, dev([0, 0, 0]), 37, cu_tokens=dev(cu))
    values = [(c.double() * s.double()[..., None, None]).cpu().numpy() for c, s in (pool.kv8_view(i, 0) for i in (0, 1))]
    run_and_compare(pool, values, tables, lens, [1, 1, 1], 4, "f16", "f16", False, q_scale=0.2)
    run_and_compare(pool, values, tables, lens, [3, 2, 5], 4, "f32", "f32", True, q_scale=0.2)
    pool.release()


def test_peaked_rows_and_unlike_scales(cuda_device):
    """Scores hundreds apart, V scales 2^40 apart from page to page: the running maxima of both carry it."""
    lens = [500, 500]
    tables, n_pages = scattered(2, lens)
    pool = KvPool(0, 1, 2, 128, n_pages, kv8="e4m3")
    values = fill(pool, 7)
    scales = pool.kv8_view(1, 0)[1]
    scales.copy_(torch.exp2(torch.randint(-30, 11, scales.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).float()))
    values[1] = (pool.kv8_view(1, 0)[0].double() * scales.double()[..., None, None]).cpu().numpy()
    run_and_compare(pool, values, tables, lens, [1, 1], 8, "f32", "f32", False, q_scale=12.0)
    run_and_compare(pool, values, tables, lens, [1, 1], 8, "f32", "f32", False, q_scale=0.001)
    run_and_compare(pool, values, tables, lens, [1, 1], 8, "f32", "f32", False, q_scale=1e30, scale=1e-31)
    pool.release()


def test_a_row_with_nan_spoils_itself_alone(cuda_device):
    lens = [40, 40]
    tables, n_pages = scattered(2, lens)
    pool = KvPool(0, 1, 2, 128, n_pages, kv8="int8")
    fill(pool, 7)
    q = torch.randn(2, 4, 128, device="cuda").half()
    ws = kv8_workspace(pool, 2, 4)
    want = kv8_attend(pool, 0, q, dev(tables), dev(lens), 40, ws)
    q2 = q.clone()
    q2[0, 1, 5], q2[1, 2, 0] = NAN, INF
    got = kv8_attend(pool, 0, q2, dev(tables), dev(lens), 40, ws)
    bad = torch.zeros(2, 4, dtype=torch.bool, device="cuda")
    bad[0, 1] = bad[1, 2] = True
    assert torch.isnan(got[bad]).all() and torch.equal(got[~bad], want[~bad])
    pool.release()


def test_same_call_same_bits(cuda_device):
    lens = [5000, 100, 2]
    tables, n_pages = scattered(2, lens)
    pool = KvPool(0, 1, 2, 256, n_pages, kv8="e4m3")
    fill(pool, 7)
    q = torch.randn(3, 16, 256, device="cuda").half()
    ws = kv8_workspace(pool, 3, 16)
    first = kv8_attend(pool, 0, q, dev(tables), dev(lens), 5000, ws)
    for _ in range(3):
        ws.random_(0, 256)
        assert torch.equal(first, kv8_attend(pool, 0, q, dev(tables), dev(lens), 5000, ws))
    pool.release()


def test_two_streams_and_two_graphs_side_by_side(cuda_device):
    """Calls with workspaces of their own on one pool at the same time, launched and replayed."""
    lens = [3000, 100]
    tables, n_pages = scattered(2, lens)
    pool = KvPool(0, 1, 2, 128, n_pages, kv8="int8")
    fill(pool, 7)
    t, n = dev(tables), dev(lens)
    qs = [torch.randn(2, 8, 128, device="cuda").half() for _ in range(2)]
    wss = [kv8_workspace(pool, 2, 8) for _ in range(2)]
    want = [kv8_attend(pool, 0, q, t, n, 3000, w) for q, w in zip(qs, wss)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [torch.zeros_like(w) for w in want]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                kv8_attend(pool, 0, qs[i], t, n, 3000, wss[i], out=outs[i])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    graphs = []
    for i in range(2):
        outs[i].zero_()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            kv8_attend(pool, 0, qs[i], t, n, 3000, wss[i], out=outs[i])
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    pool.check()
    pool.release()


@pytest.mark.parametrize("dt", ["f16", "f32"])
def test_out_in_place_of_q(cuda_device, dt):
    """Whole units, cut ones, several passes of rows, a sequence without cells: the same bits as beside q."""
    lens = [5000, 0, 33, 700]
    tables, n_pages = scattered(5, lens)
    pool = KvPool(0, 1, 2, 128, n_pages, kv8="e4m3")
    fill(pool, 21)
    t, n = dev(tables), dev(lens)
    for n_head, max_q in ((8, 1), (16, 9)):   # 4 rows a unit; 72: three passes
        q = torch.randn(4 * max_q, n_head, 128, device="cuda").to(DTYPES[dt])
        ws = kv8_workspace(pool, 4, n_head, max_q)
        want = kv8_attend(pool, 0, q, t, n, 5000, ws, max_q=max_q)
        assert kv8_attend(pool, 0, q, t, n, 5000, ws, max_q=max_q, out=q) is q
        assert torch.equal(q, want)
    with pytest.raises(BrcError):
        wide = torch.zeros(5, 8, 128, device="cuda")
        kv8_attend(pool, 0, wide[:4], t, n, 5000, kv8_workspace(pool, 4, 8), out=wide[1:])
    for gate, stride in ((torch.ones(4 * 8 * 128 - 1, device="cuda"), 128), (torch.ones(4, 8, 128, device="cuda"), 256)):
        with pytest.raises(BrcError):
            kv8_attend(pool, 0, wide[:4], t, n, 5000, kv8_workspace(pool, 4, 8), gate=gate, gate_head_stride=stride)
    pool.check()
    pool.release()


def test_scores_of_any_size(cuda_device):
    """Scores near either end of f32, all cells alike: their mean, whatever the score.  (The sums are exact up to f32 roundings of 40 equal
    weights; a weight is exactly 2^7.)"""
    pool = KvPool(0, 1, 2, 128, 3, kv8="int8")
    t, n = dev([[0, 1, 2]]), dev([40])
    k = torch.full((40, 2, 128), 2.0 ** 60, device="cuda")
    v = torch.randint(-100, 100, (40, 2, 128), device="cuda").float()
    v[:, :, 0] = 100.0   # the scale: 1 in every page
    kv8_append(pool, 0, k, v, t, dev([0]), 40, 40)
    want = v.double().mean(0)
    ws = kv8_workspace(pool, 1, 2)
    for size in (0.0, 2.0 ** -100, 2.0 ** 20, 2.0 ** 50, 2.0 ** 59):   # q . k up to 2^126
        for sign in (1.0, -1.0):
            q = torch.full((1, 2, 128), sign * size, device="cuda")
            out = kv8_attend(pool, 0, q, t, n, 40, ws, scale=1.0)
            # 40 additions on either side of the division and three more roundings, of sums of |v| <= 100
            assert (out[0].double() - want).abs().max() <= 100 * 83 * 2.0 ** -24, (size, sign)
    pool.check()
    pool.release()


def test_outputs_belong_to_the_stream_that_writes_them(cuda_device):
    """An output made for a call on another stream must not come from memory that the current stream may still use."""
    pool = KvPool(0, 1, 2, 128, 4, kv8="int8")
    fill(pool, 3)
    t, n, zero = dev([[0, 1]]), dev([20]), dev([0])
    q, ws, rope, pos = torch.randn(1, 4, 128, device="cuda"), kv8_workspace(pool, 1, 4), Rope(128), dev([5])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for call in (lambda: kv8_read(pool, 0, t, zero, 20, 20, stream=side)[0], lambda: kv8_attend(pool, 0, q, t, n, 20, ws, stream=side),
                 lambda: rope.apply(q, None, pos, stream=side)[0]):
        out = call()
        shape, where = out.shape, out.data_ptr()
        side.synchronize()
        del out
        with torch.cuda.stream(side):
            back = call()                     # the block that was just given up: it is the side stream's
        assert back.data_ptr() == where
        del back
        here = [torch.empty(shape, dtype=dt, device="cuda") for dt in (torch.float16, torch.float32) for _ in range(4)]
        assert all(x.data_ptr() != where for x in here)
    torch.cuda.synchronize()
    pool.check()
    pool.release()


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_a_serving_run(cuda_device, code):
    """Prompt, decode steps and drafts with a roll-back, together as an engine uses them: q and K rotated, K and V written
    quantised, attention over the pages, then a fork that goes its own way."""
    n_head, n_kv, hd = 8, 2, 128
    tables, n_pages = scattered(1, [200, 200], spare=6)
    pool = KvPool(0, 1, n_kv, hd, n_pages, kv8=code)
    pool.alloc(n_pages)
    pool.release_pages(np.setdiff1d(np.arange(n_pages), tables))   # the tables' pages stay held
    rope = Rope(64, theta=500000.0, scaling="bands", factor=8.0, orig_ctx=8192)
    freqs = ref.rope_freqs(64, 500000.0, "bands", 8.0, 8192)
    g = torch.Generator(device="cuda").manual_seed(6)
    t, ws = dev(tables), kv8_workspace(pool, 2, n_head, 4)
    lens, big = np.array([0, 0]), 0.0
    exact = [[np.zeros((0, n_kv, hd))] * 2 for _ in range(2)]   # unquantised keys and values, in 64 bits
    for counts, keep in (([90, 31], [90, 31]), ([1, 1], [1, 1]), ([4, 3], [2, 1]), ([1, 4], [1, 4]), ([1, 1], [1, 1])):
        total, cu = sum(counts), np.concatenate([[0], np.cumsum(counts)])
        q = torch.randn(total, n_head, hd, device="cuda", generator=g)
        k, v = (torch.randn(total, n_kv, hd, device="cuda", generator=g) for _ in range(2))
        pos = np.concatenate([np.arange(p, p + n) for p, n in zip(lens, counts)])
        qr, _ = rope.apply(q, None, dev(pos))
        kv8_append(pool, 0, k, v, t, dev(lens), int((lens + counts).max()), cu_tokens=dev(cu), rope=rope)
        kn, vn = ref.rotate(k.double().cpu().numpy(), pos, freqs, "half"), v.double().cpu().numpy()
        now = [[np.concatenate([exact[s][0], kn[cu[s]:cu[s + 1]]]), np.concatenate([exact[s][1], vn[cu[s]:cu[s + 1]]])] for s in range(2)]
        big = max(big, np.abs(kn).max(), np.abs(vn).max())
        held = []
        for s in range(2):
            n = int(lens[s]) + counts[s]
            held.append([x.double().cpu().numpy() for x in kv8_read(pool, 0, dev(tables[s:s + 1]), dev([0]), n, tokens_per_seq=n, dtype=torch.float32)])
        if max(counts) <= 4:
            out = kv8_attend(pool, 0, qr, t, dev(lens + counts), int((lens + counts).max()), ws, max_q=max(counts), cu_q=dev(cu))
            qn = ref.rotate(q.double().cpu().numpy(), pos, freqs, "half")
            for s in range(2):
                for i in range(counts[s]):
                    n = int(lens[s]) + i + 1
                    row = out[cu[s] + i].double().cpu().numpy()
                    # against the cache's own values: q's rotation in f32 (a few 2^-24 of it into the scores), the sums in f32
                    want, mag, dot = ref.attention(qn[cu[s] + i], *held[s], n, 1 / math.sqrt(hd))
                    assert (np.abs(row - want) <= mag * 2.0 ** -17 * (1 + dot[:, None])).all()
                    # against what was put in: half a step of the codes on K and V, e4m3 2^-4 of each value (below the least normal code 2^-10 of a
                    # scale), int8 half a scale, at most big / 127; rounded again each time the scale doubles or more: twice that
                    # in all.  K's enters the exponent twice (score and normaliser)
                    want, mag, dot = ref.attention(qn[cu[s] + i], now[s][0], now[s][1], n, 1 / math.sqrt(hd))
                    eps = 2.0 ** -4 if code == "e4m3" else None
                    dk = eps * dot.max() if eps else 2 * big / 127 * np.abs(qn[cu[s] + i]).sum(-1).max() / math.sqrt(hd)
                    tol = mag * (np.exp(2 * dk) - 1) + (2 * eps * mag if eps else 4 * big / 127) + 1e-3
                    assert (np.abs(row - want) <= tol).all()
        exact = [[x[: int(lens[s]) + keep[s]] for x in now[s]] for s in range(2)]
        lens = lens + keep
    pool.check()
    child, fresh = pool.fork(tables[0][: -(-int(lens[0]) // 16)], int(lens[0]))
    row = np.zeros_like(tables[0])
    row[: len(child)] = child
    both = kv8_read(pool, 0, dev(np.stack([tables[0], row])), dev([0, 0]), int(lens[0]), tokens_per_seq=int(lens[0]), dtype=torch.float32)
    n = int(lens[0])
    assert fresh is not None and all(torch.equal(x[:n], x[n:]) for x in both)
    one = torch.full((1, n_kv, hd), 1e3, device="cuda")
    kv8_append(pool, 0, one, one, dev(row[None]), dev([n]), n + 1)
    again = kv8_read(pool, 0, dev(tables[:1]), dev([0]), n, tokens_per_seq=n, dtype=torch.float32)
    assert all(torch.equal(a, b[:n]) for a, b in zip(again, both))
    pool.check()
    pool.release()


def test_the_decode_batch_of_such_a_pool(cuda_device):
    """DecodeBatch.append / attend (brc_kv_append, brc_paged_decode_attn) take an 8-bit pool."""
    lens = np.array([100, 17, 64])
    tables, n_pages = scattered(1, lens + 2)
    pool = KvPool(0, 2, 2, 256, n_pages, kv8="e4m3")
    fill(pool, 1, layer=1)
    batch = DecodeBatch(pool, 16, tables, lens, q_dtype=_lib.DTYPE_F16)
    k, v = torch.randn(3, 512, device="cuda"), torch.randn(3, 512, device="cuda")
    q = torch.randn(3, 16, 256, device="cuda").half()
    gate = torch.randn(3, 16, 512, device="cuda")
    out = torch.empty(3, 16, 256, device="cuda")
    batch.begin_step()
    batch.append(1, k, v)
    batch.attend(1, q, out, gate.view(-1)[256:], 512)
    pool.check()
    want = kv8_attend(pool, 1, q, dev(tables), dev(lens + 1), 101, kv8_workspace(pool, 3, 16), out_dtype=torch.float32, gate=gate.view(-1)[256:],
                      gate_head_stride=512)
    assert torch.equal(out, want)
    got, _ = kv8_read(pool, 1, dev(tables), dev(lens), 101, dtype=torch.float32)
    assert (got.view(3, 512) - k).abs().max() <= 2.0 ** -4 * k.abs().max()
    pool.release()


def test_pages_travel_with_their_scales(cuda_device, tmp_path):
    """Whole-page copies and the host tier carry codes and scales; a cold store refuses pages of the other code."""
    import ctypes as C

    pool = KvPool(0, 2, 2, 128, 8, kv8="e4m3")
    for layer in (0, 1):
        fill(pool, 3 + layer, layer)
    before = [[x.clone() for x in pool.kv8_view(s, l)] for s in (0, 1) for l in (0, 1)]
    ids = pool.alloc(4)
    pool.copy_pages([ids[1]], [ids[3]])
    after = [pool.kv8_view(s, l) for s in (0, 1) for l in (0, 1)]
    for a, b in zip(after, before):
        assert all(torch.equal(x[int(ids[3])].float(), y[int(ids[1])].float()) for x, y in zip(a, b))
    tier = C.c_void_p()
    _lib.call("brc_tier_create", pool.handle, 4, C.byref(tier))
    page, slot, back = (C.c_uint32 * 1)(int(ids[1])), (C.c_uint32 * 1)(), (C.c_uint32 * 1)()
    _lib.call("brc_tier_demote", tier, page, 1, slot, None)
    _lib.call("brc_tier_sync", tier)
    pool.zero()
    torch.cuda.synchronize()
    _lib.call("brc_tier_promote", tier, slot, 1, back)
    _lib.call("brc_tier_sync", tier)
    for a, b in zip(after, before):
        assert all(torch.equal(x[back[0]].float(), y[int(ids[1])].float()) for x, y in zip(a, b))
    cold = C.c_void_p()
    path = str(tmp_path / "cold").encode()
    _lib.call("brc_cold_open", tier, path, 2, 1, C.byref(cold))
    _lib.call("brc_cold_close", cold)
    other = KvPool(0, 2, 2, 128, 8, kv8="int8")
    tier2 = C.c_void_p()
    _lib.call("brc_tier_create", other.handle, 4, C.byref(tier2))
    assert _lib.load().brc_cold_open(tier2, path, 0, 0, C.byref(cold)) == _lib.ERR_INVALID
    for x in (tier, tier2):
        _lib.call("brc_tier_destroy", x)
    pool.release()
    other.release()


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("n_head,n_kv,hd,max_q", [(16, 2, 256, 1), (6, 3, 128, 1), (16, 2, 256, 2), (8, 2, 128, 9)])
def test_sixteen_bit_results_are_rounded_once(cuda_device, code, dt, n_head, n_kv, hd, max_q):
    """16-bit q and out: the result is the f32 one rounded to the type, its weights not rounded to 16 bits in front of that.

    Scores near one another (q small), so that the exponent's own error is small and weights lie just under a power of two, where a
    weight in one binary16 part would be off by up to 2^-12 of itself; two parts: 2^-22.  Few cells, and columns where values cancel."""
    lens = [2, 3, 5, 9, 16, 17, 40, 300]
    tables, n_pages = scattered(2, lens)
    pool = KvPool(0, 1, n_kv, hd, n_pages, kv8=code)
    values = fill(pool, 3)
    q = (torch.randn(len(lens) * max_q, n_head, hd, device="cuda", generator=torch.Generator(device="cuda").manual_seed(4)) * 0.05).to(DTYPES[dt])
    got = kv8_attend(pool, 0, q, dev(tables), dev(lens), max(lens), kv8_workspace(pool, len(lens), n_head, max_q), max_q=max_q)
    pool.check()
    assert got.dtype == DTYPES[dt]
    got, qn, fi = got.double().cpu().numpy(), q.double().cpu().numpy(), torch.finfo(DTYPES[dt])
    for s, n in enumerate(lens):
        k, v = (cells(x, tables[s], n) for x in values)
        for i in range(max_q):
            want, mag, dot = ref.attention(qn[s * max_q + i], k, v, n - (max_q - 1 - i), 1 / math.sqrt(hd))
            # as in run_and_compare with the two parts' 2^-22 on numerator and denominator; below the second part's range half binary16's
            # least spacing, 2^-25 beside a heaviest weight of 2^7 or more, for each cell; then out's half step
            exponent = 2 * (hd / 16 + 4) * 2.0 ** -22 * dot[:, None] + 4 * 2.0 ** -21
            tol = mag * (2.0 ** -21 + 2 * exponent + 2 * (n / 16 + 32) * 2.0 ** -22) + n * 2.0 ** -32 * np.abs(v).max()
            tol = tol * (1 + fi.eps) + fi.eps / 2 * np.abs(want) + fi.tiny * fi.eps
            err = np.abs(got[s * max_q + i] - want)
            assert (err <= tol).all(), (s, i, float((err - tol).max()), float(err.max()))
    pool.release()


@pytest.mark.parametrize("n_head,max_q", [(8, 4), (40, 4)])   # 16 rows; 80: three passes
def test_a_prefix_that_leads_past_the_rows(cuda_device, n_head, max_q):
    """cu_q of another step: rows that q and out do not have are neither read nor written, a prefix that goes backwards is no rows; both
    reported, and what is there is as it would be."""
    lens = [700, 90, 33]
    tables, n_pages = scattered(5, lens)
    pool = KvPool(0, 1, 2, 128, n_pages, kv8="int8")
    fill(pool, 3)
    ws, big = kv8_workspace(pool, 3, n_head, max_q), torch.randn(12, n_head, 128, device="cuda")

    def call(rows, cu):
        q, out = big.clone(), torch.full_like(big, 7.0)
        q[rows:] = NAN
        kv8_attend(pool, 0, q[:rows], dev(tables), dev(lens), 700, ws, max_q=max_q, cu_q=dev(cu), out=out[:rows])
        return out

    want = call(10, [0, 4, 6, 10])
    pool.check()
    assert (want[10:] == 7).all() and torch.isfinite(want[:10]).all()
    for rows, cu, live in ((8, [0, 4, 6, 10], 8), (5, [0, 4, 6, 10], 5), (10, [0, 4, 6, 2 ** 31 - 1], 6), (8, [0, 4, 9, 12], 4), (6, [0, 4, 2, 2], 4)):
        got = call(rows, cu)
        with pytest.raises(BrcError, match="position past bound"):
            pool.check()
        # f32 sums in another order where the cut moved: far apart only if a row saw other cells
        assert torch.allclose(got[:live], want[:live], rtol=1e-4, atol=1e-4) and (got[rows:] == 7).all()
    pool.check()
    pool.release()


def test_a_ragged_batch_without_tokens(cuda_device):
    """No sequence has a token this step: an empty q (whose address is 0) is an empty result, as in the append."""
    pool = KvPool(0, 1, 2, 128, 4, kv8="int8")
    t, lens, cu, q = dev([[0], [1], [2]]), dev([3, 16, 0]), dev([0, 0, 0, 0]), torch.ones(0, 8, 128, device="cuda")
    assert kv8_attend(pool, 0, q, t, lens, 16, kv8_workspace(pool, 3, 8, 4), max_q=4, cu_q=cu).shape == (0, 8, 128)
    with pytest.raises(BrcError):
        kv8_attend(pool, 1, q, t, lens, 16, kv8_workspace(pool, 3, 8, 4), max_q=4, cu_q=cu)   # checked all the same
    pool.check()
    pool.release()


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("dt", ["f16", "f32"])
@pytest.mark.parametrize("n_head,n_kv,hd,n_q", [(40, 2, 128, [1, 1, 8, 0, 1, 3, 1, 8]), (16, 2, 256, [1, 9, 1, 0, 4, 1, 5, 1]), (5, 1, 256, [0, 1, 0, 16, 7, 1, 2, 1])])
def test_sequences_take_the_passes_of_their_own_rows(cuda_device, code, dt, n_head, n_kv, hd, n_q):
    tables, n_pages = scattered(2, LENS)
    pool = KvPool(0, 1, n_kv, hd, n_pages, kv8=code)
    values = fill(pool, 4)
    run_and_compare(pool, values, tables, LENS, n_q, n_head, dt, dt, True, gate=True)
    pool.release()


def test_short_drafts_beside_a_long_one_stream_their_cache_once(cuda_device):
    """One sequence of 8 tokens (160 rows, five passes) beside 31 of one (20 rows, one pass): close to a call of 32 sequences of one token
    (36 streams against 32), and far from five passes for everybody (160 against 32)."""
    n, cells_each, n_head = 32, 16384, 40
    pool = KvPool(0, 1, 2, 128, n * cells_each // 16, kv8="int8")
    tables, lens = dev(np.arange(n * cells_each // 16).reshape(n, -1)), dev([cells_each] * n)
    n_q = [1] * (n - 1) + [8]
    q, ws = torch.randn(sum(n_q), n_head, 128, device="cuda").half(), kv8_workspace(pool, n, n_head, 8)

    def ms(call):
        times = []
        for _ in range(9):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            torch.cuda._sleep(200_000)      # the call is issued while the GPU is still busy
            a.record()
            call()
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        return sorted(times)[4]

    cu = dev(np.concatenate([[0], np.cumsum(n_q)]))
    one = ms(lambda: kv8_attend(pool, 0, q[:n], tables, lens, cells_each, ws))
    mixed = ms(lambda: kv8_attend(pool, 0, q, tables, lens, cells_each, ws, max_q=8, cu_q=cu))
    assert mixed < 2.2 * one, (one, mixed)   # geometric middle of 36 / 32 and 160 / 32: 2.4
    pool.check()
    pool.release()


def test_gates_of_any_size(cuda_device):
    """One cell, whose weight is 1: v times the gate's sigmoid, from closed gates (denormal) to open ones."""
    pool = KvPool(0, 1, 2, 128, 1, kv8="int8")
    fill(pool, 3)
    v = (pool.kv8_view(1, 0)[0].double() * pool.kv8_view(1, 0)[1].double()[..., None, None])[0, :, 0].repeat_interleave(4, 0)   # [8 heads][128]
    gate = torch.linspace(-104, 104, 8 * 128, device="cuda").view(1, 8, 128)
    gate[0, 0, 0], gate[0, 7, 127] = -INF, INF
    q = torch.randn(1, 8, 128, device="cuda")
    out = kv8_attend(pool, 0, q, dev([[0]]), dev([1]), 16, kv8_workspace(pool, 1, 8), gate=gate, gate_head_stride=128)[0].double()
    want = v * torch.sigmoid(gate[0].double())
    # two exponentials of base 2 and a division in front of the gate (2^-21 each at most, ex2.approx' bound), then expf (an ulp or two: 2^-22),
    # a sum, a quotient and a product of half a step each; at the denormal end a step of 2^-149 in the sigmoid and one in the product
    tol = want.abs() * (3 * 2.0 ** -21 + 2.0 ** -21) + (v.abs() + 1) * 2.0 ** -148
    assert ((out - want).abs() <= tol).all(), ((out - want).abs() - tol).max()
    pool.check()
    pool.release()


def test_what_check_says_of_an_infinity(cuda_device):
    """The write took place, so no index was refused; beside a refused one both are named."""
    pool = KvPool(0, 1, 2, 128, 2, kv8="int8")
    k = torch.ones(20, 2, 128, device="cuda")
    k[17, 1, 3] = INF
    kv8_append(pool, 0, k, k, dev([[0, 1]]), dev([0]), 20, tokens_per_seq=20)
    with pytest.raises(BrcError, match="infinity or NaN reached a quantising write, which stored") as e:
        pool.check()
    assert "refused" not in str(e.value) and "row 16" in str(e.value)   # the first row of its page
    kv8_append(pool, 0, k, k, dev([[7, 1]]), dev([0]), 20, tokens_per_seq=20)
    with pytest.raises(BrcError, match="refused an index.*page id.*infinity or NaN"):
        pool.check()
    pool.check()
    pool.release()


@pytest.mark.parametrize("n_seqs,n_kv,hd,dtype,n", [(160, 5, 128, "bf16", 1), (70, 8, 128, "f16", 1), (150, 2, 256, "f32", 1), (1, 7, 128, "f16", 3000), (300, 3, 128, "bf16", 2)])
def test_append_with_some_heads_a_cta(cuda_device, n_seqs, n_kv, hd, dtype, n):
    """Calls whose heads are dealt out in groups, the last one smaller: every head once, kept cells in front of the new ones."""
    g = torch.Generator(device="cuda").manual_seed(2)
    first = np.random.default_rng(1).integers(1, 15, n_seqs)
    tables, n_pages = scattered(3, first + n)
    pool, cache = KvPool(0, 1, n_kv, hd, n_pages, kv8="e4m3"), ref.Cache(n_pages, n_kv, hd, "e4m3")
    pool.poison_nan()
    at, t = np.zeros(n_seqs, np.int64), dev(tables)
    for counts in (first, np.full(n_seqs, n)):
        cu = np.concatenate([[0], np.cumsum(counts)])
        k, v = (random_rows(g, int(cu[-1]), n_kv, hd, dtype) for _ in range(2))
        kv8_append(pool, 0, k, v, t, dev(at), int((at + counts).max()), cu_tokens=dev(cu))
        kn, vn = k.double().cpu().numpy(), v.double().cpu().numpy()
        for s in range(n_seqs):
            cache.append(tables[s], int(at[s]), kn[cu[s]:cu[s + 1]], vn[cu[s]:cu[s + 1]])
        at += counts
    pool.check()
    assert_pool_is(pool, cache, tables, at)
    pool.release()


def rotation_error(x, m=1.0):
    """test_rope_gpu.tolerance: f32 arithmetic on a pair, 8 * 2^-24 * 2 max|x| m."""
    return 8 * 2.0 ** -24 * 2 * np.abs(x).max() * m


def code_steps(x, scale, code):
    """Distance between neighbouring codes around x, in x's units."""
    return ref.step_of(x / scale, code) * scale


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout,n_rot,offset", [("half", 256, 0), ("half", 64, 0), ("half", 90, 0), ("half", 128, 1), ("interleaved", 256, 0), ("interleaved", 90, 1)])
def test_append_rotates_keys_of_256(cuda_device, code, dtype, layout, n_rot, offset):
    """Heads of 256, whose rows are half a block: every pairing, aligned and not, one token and chunks; V as it comes."""
    n_kv, hd = 2, 256
    counts, pos0 = [40, 1, 19], [70003, 16, 5]
    own, n_pages = scattered(5, [p % 16 + n for p, n in zip(pos0, counts)])
    wide = np.zeros((3, max(pos0) // 16 + own.shape[1]), np.int32)
    for s, p in enumerate(pos0):
        wide[s, p // 16:p // 16 + own.shape[1]] = own[s]
    g = torch.Generator(device="cuda").manual_seed(2)
    total, row = sum(counts), 2 * n_kv * hd + offset
    m = torch.randn(total * row + offset, device="cuda", generator=g).to(DTYPES[dtype])[offset:].view(total, row)
    pool = KvPool(0, 1, n_kv, hd, n_pages, kv8=code)
    rope = Rope(n_rot, theta=500000.0, layout=layout, scaling="yarn", factor=16.0, orig_ctx=8192)
    cu, end = np.concatenate([[0], np.cumsum(counts)]), max(p + n for p, n in zip(pos0, counts))
    kv8_append(pool, 0, m[:, :n_kv * hd], m[:, n_kv * hd:2 * n_kv * hd], dev(wide), dev(pos0), end, cu_tokens=dev(cu), rope=rope)
    got = [x.double().cpu().numpy() for x in kv8_read(pool, 0, dev(wide), dev(pos0), end, cu_tokens=dev(cu), total_tokens=total, dtype=torch.float32)]
    pool.check()
    pos = np.concatenate([np.arange(p, p + n) for p, n in zip(pos0, counts)])
    rows = m.double().cpu().numpy()
    xk = ref.rotate(rows[:, :n_kv * hd].reshape(total, n_kv, hd), pos, ref.rope_freqs(n_rot, 500000.0, "yarn", 16.0, 8192), layout, rope.factor)
    xv = rows[:, n_kv * hd:2 * n_kv * hd].reshape(total, n_kv, hd)
    page = np.array([wide[np.searchsorted(cu, a, "right") - 1, pos[a] // 16] for a in range(total)])
    for side, (x, fuzz) in enumerate(((xk, rotation_error(rows, rope.factor)), (xv, 0.0))):
        scale = pool.kv8_view(side, 0)[1].double().cpu().numpy()[page][:, :, None]
        # half a step; K's f32 error moves a value, and with it the border that it is rounded at
        assert (np.abs(got[side] - x) <= code_steps(x, scale, code) / 2 + 2 * fuzz).all(), np.abs(got[side] - x).max()
        for i in np.unique(page):   # and no scale larger than the page needs
            amax = np.abs(x[page == i]).max((0, 2))
            assert all(scale[page == i][0, h, 0] <= 2.0 ** ref.exponent(amax[h] + fuzz, code) for h in range(n_kv))
    pool.release()


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_a_serving_run_stores_what_was_put_in(cuda_device, code, layout):
    """Prompt, decode steps, drafts with a roll-back: after each of them every cached key and value lies within the code's rounding of the
    exact one, and keys that were not rotated, or rotated the other way about, would not."""
    n_kv, hd = 2, 128
    tables, n_pages = scattered(1, [200, 200])
    pool, t = KvPool(0, 1, n_kv, hd, n_pages, kv8=code), dev(tables)
    rope = Rope(64, theta=500000.0, layout=layout, scaling="bands", factor=8.0, orig_ctx=8192)
    freqs, g = ref.rope_freqs(64, 500000.0, "bands", 8.0, 8192), torch.Generator(device="cuda").manual_seed(6)
    lens = np.array([0, 0])
    none = np.zeros((0, n_kv, hd))
    exact = [[none, none, none, none] for _ in range(2)]                        # keys, values; keys as they came, keys by the other layout
    written = [[np.zeros((0, n_kv, 1))] * 2 for _ in range(2)]                  # each cell's scale when it was written
    for counts, keep in (([90, 31], [90, 31]), ([1, 1], [1, 1]), ([4, 3], [2, 1]), ([1, 4], [1, 4]), ([20, 1], [20, 1]), ([1, 1], [1, 1])):
        cu = np.concatenate([[0], np.cumsum(counts)])
        k, v = (random_rows(g, int(cu[-1]), n_kv, hd, "f32") for _ in range(2))
        pos = np.concatenate([np.arange(p, p + n) for p, n in zip(lens, counts)])
        kv8_append(pool, 0, k, v, t, dev(lens), int((lens + counts).max()), cu_tokens=dev(cu), rope=rope)
        pool.check()
        raw = k.double().cpu().numpy()
        new = [ref.rotate(raw, pos, freqs, layout), v.double().cpu().numpy(), raw, ref.rotate(raw, pos, freqs, "half" if layout == "interleaved" else "interleaved")]
        fuzz = rotation_error(raw)
        for s in range(2):
            n = int(lens[s]) + counts[s]
            now = [np.concatenate([a, b[cu[s]:cu[s + 1]]]) for a, b in zip(exact[s], new)]
            held = [x.double().cpu().numpy() for x in kv8_read(pool, 0, dev(tables[s:s + 1]), dev([0]), n, tokens_per_seq=n, dtype=torch.float32)]
            for side in (0, 1):
                scale = pool.kv8_view(side, 0)[1].double().cpu().numpy()[tables[s][np.arange(n) // 16]][:, :, None]
                written[s][side] = np.concatenate([written[s][side], scale[int(lens[s]):]])
                # half a step of the present scale; a cell whose page has grown since was rounded at every smaller scale too: half a step of
                # each, together at most another half of the present one
                room = code_steps(now[side], scale, code) * np.where(scale > written[s][side], 1.0, 0.5) + (2 * fuzz if side == 0 else 0.0)
                assert (np.abs(held[side] - now[side]) <= room).all(), (side, s, counts)
                if side == 0 and n > 40:
                    for wrong in now[2:]:
                        assert (np.abs(held[0] - wrong) > code_steps(wrong, scale, code) + 2 * fuzz).mean() > 0.05
            exact[s] = [x[: int(lens[s]) + keep[s]] for x in now]
            written[s] = [x[: int(lens[s]) + keep[s]] for x in written[s]]
        lens = lens + keep
    pool.release()
