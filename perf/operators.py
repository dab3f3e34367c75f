"""Cases of the 8-bit cache operators: rotary positions, the quantising write with its read-back, and attention.

Where `own` is false, run() computes the operators in plain torch; where it is true it calls the framework.

An 8-bit cache page holds 16 cells.  Per page, kv head and side (K or V) it has codes [16][head_dim] (e4m3 or int8) and one
scale, a power of two: the least with max|x| / scale <= 448 (e4m3) or 127 (int8) over what was written.  A write into a
page that already holds cells keeps the larger of the old and the needed scale and rounds the kept codes to it again.
"""
import math
import random

import torch

own = False

CELLS = 16
DEV = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
EXP_MIN, EXP_MAX = -120, 120


# ------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of 32 sequences: the new tokens' q and k, f32 as the projections give them, a quarter of the head rotated
        {"name": "rope_step", "op": "rope", "tokens": 32, "n_head": 16, "n_kv": 2, "hd": 256, "n_rot": 64, "layout": "half",
         "scaling": "none", "max_pos": 8192, "dtype": "f32"},
        # a prefill chunk of a long-context model: whole head, interleaved pairs, yarn to 131072 positions
        {"name": "rope_chunk_yarn", "op": "rope", "tokens": 16384, "n_head": 32, "n_kv": 8, "hd": 128, "n_rot": 128,
         "layout": "interleaved", "scaling": "yarn", "max_pos": 131072, "dtype": "bf16"},
        # an odd batch at far positions, wavelength bands, part of the head, half layout
        {"name": "rope_far_bands", "op": "rope", "tokens": 1001, "n_head": 16, "n_kv": 2, "hd": 256, "n_rot": 192,
         "layout": "half", "scaling": "bands", "max_pos": 1 << 20, "dtype": "f16"},
        # one decode step's write into part-filled pages, then those pages as values (what a check of the cache compares)
        {"name": "write_step_e4m3", "op": "write", "n_seqs": 32, "lo": 1, "hi": 1, "n_kv": 2, "hd": 256, "code": "e4m3",
         "dtype": "f16", "rope": False, "start": 8192},
        # a ragged prefill chunk, keys rotated on the way, read back for an attention that works in 16 bits
        {"name": "write_chunk_rope_int8", "op": "write", "n_seqs": 64, "lo": 100, "hi": 400, "n_kv": 8, "hd": 128, "code": "int8",
         "dtype": "bf16", "rope": True, "start": 5000},
        # one sequence's whole cache back in 16 bits
        {"name": "read_one_e4m3", "op": "read", "n_seqs": 1, "lo": 8190, "hi": 8190, "n_kv": 2, "hd": 256, "code": "e4m3", "dtype": "f16"},
        # a ragged batch's caches back, for a hand-over to an engine that keeps 16 bits
        {"name": "read_batch_int8", "op": "read", "n_seqs": 24, "lo": 1000, "hi": 16384, "n_kv": 8, "hd": 128, "code": "int8", "dtype": "bf16"},
        # a single short conversation
        {"name": "attend_short", "op": "attend", "n_seqs": 1, "lo": 700, "hi": 700, "q_len": 1, "ragged_q": False, "n_head": 16,
         "n_kv": 2, "hd": 256, "code": "e4m3", "dtype": "f16"},
        # the benchmark's decode batch, 32 sequences of 512 .. 8192 cells
        {"name": "attend_batch", "op": "attend", "n_seqs": 32, "lo": 512, "hi": 8192, "q_len": 1, "ragged_q": False, "n_head": 16,
         "n_kv": 2, "hd": 256, "code": "e4m3", "dtype": "f16"},
        # one long document
        {"name": "attend_long_int8", "op": "attend", "n_seqs": 1, "lo": 131072, "hi": 131072, "q_len": 1, "ragged_q": False,
         "n_head": 16, "n_kv": 2, "hd": 256, "code": "int8", "dtype": "f32"},
        # drafted tokens of 24 sequences in one pass, one to four each
        {"name": "attend_drafts_int8", "op": "attend", "n_seqs": 24, "lo": 1024, "hi": 6000, "q_len": 4, "ragged_q": True,
         "n_head": 32, "n_kv": 8, "hd": 128, "code": "int8", "dtype": "bf16"},
        # a large batch of long contexts: the cache no on-chip memory holds
        {"name": "attend_large", "op": "attend", "n_seqs": 48, "lo": 4096, "hi": 24576, "q_len": 1, "ragged_q": False, "n_head": 16,
         "n_kv": 2, "hd": 256, "code": "e4m3", "dtype": "bf16"},
    ]


def spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    n_head, n_kv, hd = rng.choice([(16, 2, 256), (24, 2, 256), (8, 1, 256), (32, 8, 128), (12, 4, 128), (7, 7, 128), (20, 5, 128), (40, 2, 128)])
    code, dtype = rng.choice(["e4m3", "int8"]), rng.choice(["f16", "bf16", "f32"])
    op = rng.choice(["rope", "write", "read", "attend", "attend"])
    if op == "rope":
        tokens = spread(rng, 1, max(1, 80_000_000 // ((n_head + n_kv) * hd)))
        return {"op": op, "tokens": tokens, "n_head": n_head, "n_kv": n_kv, "hd": hd, "n_rot": 2 * rng.randint(2, hd // 2),
                "layout": rng.choice(["half", "interleaved"]), "scaling": rng.choice(["none", "linear", "ntk", "yarn", "bands"]),
                "max_pos": spread(rng, 2048, 1 << 21), "dtype": dtype}
    if op == "write":
        n_seqs = spread(rng, 1, 64)
        hi = spread(rng, 1, max(1, 16000 // n_seqs))
        # read back in 16 bits: an 8-bit code on the border between two roundings may go either way after a rotation in 32 bits
        return {"op": op, "n_seqs": n_seqs, "lo": spread(rng, 1, hi), "hi": hi, "n_kv": n_kv, "hd": hd, "code": code,
                "dtype": rng.choice(["f16", "bf16"]), "rope": rng.random() < 0.5, "start": spread(rng, 1, 9000)}
    cells = 200_000_000 // (n_kv * hd)
    n_seqs = spread(rng, 1, 48)
    hi = min(131072, spread(rng, 1, max(1, cells // n_seqs)))
    lo = spread(rng, 1, hi)
    if op == "read":
        return {"op": op, "n_seqs": n_seqs, "lo": lo, "hi": hi, "n_kv": n_kv, "hd": hd, "code": code, "dtype": dtype}
    q_len = rng.choice([1, 1, 1, 2, 3, 4, 6, 8])
    return {"op": op, "n_seqs": n_seqs, "lo": lo, "hi": hi, "q_len": q_len, "ragged_q": rng.random() < 0.5, "n_head": n_head, "n_kv": n_kv,
            "hd": hd, "code": code, "dtype": dtype}


def lengths(case):
    """The sequences' lengths (cells, or tokens to write): the case's alone, so that work() knows them."""
    r = random.Random(case["n_seqs"] * 1000003 + case["lo"] * 1009 + case["hi"])
    return [r.randint(case["lo"], case["hi"]) for _ in range(case["n_seqs"])]


def q_lengths(case):
    r = random.Random(case["n_seqs"] * 7919 + case["q_len"])
    return [r.randint(1, case["q_len"]) if case["ragged_q"] else case["q_len"] for _ in range(case["n_seqs"])]


def starts(case):
    """Where a write begins in each sequence."""
    r = random.Random(case["start"] * 31 + case["n_seqs"])
    return [r.randint(0, case["start"]) for _ in range(case["n_seqs"])]


def pages_of(cells):
    return -(-cells // CELLS)


def work(case):
    op = case["op"]
    if op == "rope":
        values = case["tokens"] * (case["n_head"] + case["n_kv"]) * case["hd"]
        return {"bytes": 2 * values * DTYPES[case["dtype"]].itemsize + 4 * case["tokens"], "flops": 3 * values * case["n_rot"] // case["hd"]}
    row = case["n_kv"] * case["hd"]
    size = DTYPES[case["dtype"]].itemsize
    if op == "write":
        total, back = 0, 0
        for n, p in zip(lengths(case), starts(case)):
            total += n
            back += n + p % CELLS
        # source read, codes written; codes read and values written by the read-back
        return {"bytes": 2 * (total * row * (size + 1) + back * row * (size + 1)), "flops": 4 * (total + back) * row}
    cells = sum(lengths(case))
    scales = sum(pages_of(n) for n in lengths(case)) * case["n_kv"] * 8
    if op == "read":
        return {"bytes": 2 * cells * row * (1 + size) + scales, "flops": 2 * cells * row}
    ql = q_lengths(case)
    flops = sum(4 * n * t * case["n_head"] * case["hd"] for n, t in zip(lengths(case), ql))
    return {"bytes": 2 * cells * row + scales + 2 * sum(ql) * case["n_head"] * case["hd"] * size, "flops": flops}


# ------------------------------------------------------------------------------------------------- what a user has in hand
ROPE = {"none": {}, "linear": {"factor": 4.0}, "ntk": {"factor": 8.0}, "yarn": {"factor": 16.0, "orig_ctx": 8192},
        "bands": {"factor": 8.0, "orig_ctx": 8192}}
THETA = 500000.0


def rope_freqs(n_rot, scaling, theta=THETA):
    """Angle per position of each pair, float64, and the factor on the rotated values."""
    a = ROPE[scaling]
    j = torch.arange(0, n_rot, 2, dtype=torch.float64, device=DEV)
    if scaling == "ntk":
        theta = theta * a["factor"] ** (n_rot / (n_rot - 2))
    f = theta ** (-j / n_rot)
    if scaling == "linear":
        return f / a["factor"], 1.0
    if scaling == "yarn":
        at = [n_rot * math.log(a["orig_ctx"] / (b * 2 * math.pi)) / (2 * math.log(theta)) for b in (32.0, 1.0)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), n_rot - 1)
        ramp = ((j / 2 - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return f / a["factor"] * ramp + f * (1 - ramp), 0.1 * math.log(a["factor"]) + 1
    if scaling == "bands":
        turns = a["orig_ctx"] * f / (2 * math.pi)
        smooth = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return (1 - smooth) * f / a["factor"] + smooth * f, 1.0
    return f, 1.0


def rope_plan(n_rot, layout, scaling):
    if own:
        from breccia_b200.qsa import Rope

        return Rope(n_rot, theta=THETA, layout=layout, scaling=scaling, **ROPE[scaling])
    f, m = rope_freqs(n_rot, scaling)
    return {"n_rot": n_rot, "layout": layout, "freqs": f, "m": m}


def generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def tables(case, cells, g):
    """Scattered pages for sequences of `cells` cells: (tables [n_seqs][stride], pages in the pool).  The last page is no sequence's."""
    need = [pages_of(n) for n in cells]
    n_pages = sum(need) + max(1, sum(need) // 16) + 1
    ids = torch.randperm(n_pages - 1, generator=g, device=DEV, dtype=torch.int32)
    t = torch.full((len(need), max(need)), n_pages - 1, dtype=torch.int32, device=DEV)
    at = torch.tensor([0] + need, device=DEV).cumsum(0)
    col = torch.arange(max(need), device=DEV)
    live = col[None, :] < torch.tensor(need, device=DEV)[:, None]
    t[live] = ids[(at[:-1, None] + col[None, :])[live]]
    return t, n_pages


def make_cache(case, n_pages, g):
    """A pool's content: tokens of unlike size from head to head and page to page, quantised page by page."""
    n_kv, hd = case["n_kv"], case["hd"]
    out = []
    for _ in range(2):
        codes = torch.empty((n_pages, n_kv, CELLS, hd), dtype=CODES[case["code"]], device=DEV)
        scales = torch.empty((n_pages, n_kv), device=DEV)
        step = max(1, (1 << 26) // (n_kv * CELLS * hd))
        for i in range(0, n_pages, step):
            n = min(step, n_pages - i)
            x = randn(g, n, n_kv, CELLS, hd) * torch.exp(0.3 * randn(g, n, n_kv, 1, 1))
            scales[i:i + n] = scale_for(x.abs().amax((2, 3)), case["code"])
            codes[i:i + n] = encode(x / scales[i:i + n, :, None, None], case["code"])
        out += [codes, scales]
    return out


def make_pool(case, n_pages, cache):
    from breccia_b200.qsa import KvPool

    pool = KvPool(0, 1, case["n_kv"], case["hd"], n_pages, kv8=case["code"])
    for which in (0, 1):
        codes, scales = pool.kv8_view(which, 0)
        codes.copy_(cache[2 * which])
        scales.copy_(cache[2 * which + 1])
    return pool


def prepare(case, seed):
    g = generator(seed)
    op = case["op"]
    dtype = DTYPES[case["dtype"]]
    s = {"op": op, "case": case, "dtype": dtype}
    if op == "rope":
        s["q"] = randn(g, case["tokens"], case["n_head"], case["hd"]).to(dtype)
        s["k"] = randn(g, case["tokens"], case["n_kv"], case["hd"]).to(dtype)
        s["positions"] = torch.randint(0, case["max_pos"], (case["tokens"],), generator=g, device=DEV, dtype=torch.int32)
        s["rope"] = rope_plan(case["n_rot"], case["layout"], case["scaling"])
        return s
    lens = lengths(case)
    if op == "write":
        p0 = starts(case)
        ends = [p + n for p, n in zip(p0, lens)]
        cells = ends
        total = sum(lens)
        s["k"] = (randn(g, total, case["n_kv"], case["hd"]) * 1.5).to(dtype)
        s["v"] = randn(g, total, case["n_kv"], case["hd"]).to(dtype)
        first = [p // CELLS * CELLS for p in p0]
        back = [e - f for e, f in zip(ends, first)]
        for name, v in (("pos0", p0), ("read0", first), ("cu", [0] + lens), ("cu_back", [0] + back)):
            t = torch.tensor(v, device=DEV, dtype=torch.int32)
            s[name] = t.cumsum(0, dtype=torch.int32) if name.startswith("cu") else t
        s |= {"total": total, "total_back": sum(back), "max_end": max(ends), "most": max(lens)}
        s["rope"] = rope_plan(case["hd"] // 2, "half", "yarn") if case["rope"] else None
    else:
        cells = lens
        s["lens"] = torch.tensor(lens, device=DEV, dtype=torch.int32)
        s["max_end"] = max(lens)
        if op == "read":
            s["pos0"] = torch.zeros_like(s["lens"])
            s["cu"] = torch.tensor([0] + lens, device=DEV, dtype=torch.int32).cumsum(0, dtype=torch.int32)
            s["total"] = sum(lens)
    s["tables"], n_pages = tables(case, cells, g)
    cache = make_cache(case, n_pages, g)
    if op == "attend":
        ql = q_lengths(case)
        s["q"] = (randn(g, sum(ql), case["n_head"], case["hd"]) * 1.5).to(dtype)
        s["max_q"] = case["q_len"]
        s["cu_q"] = torch.tensor([0] + ql, device=DEV, dtype=torch.int32).cumsum(0, dtype=torch.int32) if case["ragged_q"] else None
        s["scale"] = 1 / math.sqrt(case["hd"])
    if own:
        s["pool"] = make_pool(case, n_pages, cache)
        if op == "attend":
            from breccia_b200.qsa import kv8_workspace

            s["workspace"] = kv8_workspace(s["pool"], case["n_seqs"], case["n_head"], case["q_len"])
    else:
        s["cache"] = cache
    return s


# ------------------------------------------------------------------------------------------------- plain forms
def scale_for(amax, code):
    """The least power of two with amax / scale <= the largest code."""
    top = 448.0 if code == "e4m3" else 127.0
    m, e = torch.frexp(amax.float() / top)          # amax / top = m 2^e, m in [0.5, 1): rounding cannot pass a power of two here
    e = torch.where(m > 0.5, e, e - 1)
    e = torch.where(amax * torch.exp2(-e.float()) > top, e + 1, e)
    return torch.exp2(e.clamp(EXP_MIN, EXP_MAX).float())


def encode(x, code):
    if code == "e4m3":
        return x.clamp(-448, 448).to(torch.float8_e4m3fn)
    return x.round().clamp(-127, 127).to(torch.int8)


def rotate(x, positions, plan):
    """x [tokens][heads][hd] -> f32."""
    n, half = plan["n_rot"], plan["n_rot"] // 2
    angle = positions.double()[:, None] * plan["freqs"][None, :]
    c, s = (angle.cos() * plan["m"]).float()[:, None, :], (angle.sin() * plan["m"]).float()[:, None, :]
    x = x.float()
    r, rest = x[..., :n], x[..., n:]
    if plan["layout"] == "half":
        a, b = r[..., :half], r[..., half:]
        return torch.cat([a * c - b * s, a * s + b * c, rest], -1)
    a, b = r[..., 0::2], r[..., 1::2]
    return torch.cat([torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2), rest], -1)


def token_cells(cu, pos0, total):
    """Sequence and cell of each token of a ragged batch."""
    t = torch.arange(total, device=DEV, dtype=torch.int32)
    seq = torch.searchsorted(cu, t, right=True) - 1
    return seq, pos0[seq] + t - cu[seq]


def plain_read(codes, scales, table, cu, pos0, total, dtype):
    seq, cell = token_cells(cu, pos0, total)
    page = table[seq, cell // CELLS].long()
    return (codes[page, :, cell % CELLS].float() * scales[page][:, :, None]).to(dtype)


def plain_write(codes, scales, x, s, code):
    """Every page a sequence touches at once, [n_seqs][pages]; those past its end go to the pool's spare page."""
    pos0, end = s["pos0"], s["pos0"] + s["cu"][1:] - s["cu"][:-1]
    first = pos0 // CELLS
    j = torch.arange((s["most"] + 2 * CELLS - 2) // CELLS, device=DEV)
    at = first[:, None] + j
    live = at * CELLS < end[:, None]
    table = s["tables"]
    page = torch.where(live, table.gather(1, at.clamp(max=table.shape[1] - 1).long()), codes.shape[0] - 1).long()
    cell = at[:, :, None] * CELLS + torch.arange(CELLS, device=DEV)
    new = (cell >= pos0[:, None, None]) & (cell < end[:, None, None])
    src = (s["cu"][:-1, None, None] + cell - pos0[:, None, None]).clamp(0, s["total"] - 1).long()
    tile = (x[src].float() * new[..., None, None]).transpose(2, 3)               # [n_seqs][pages][n_kv][16][hd]
    need = scale_for(tile.abs().amax((3, 4)), code)
    kept = ((cell < pos0[:, None, None]) & (j == 0)[None, :, None])
    has = kept.any(-1)[..., None]
    old = scales[page]
    scale = torch.where(has, torch.maximum(need, old), need)
    held = codes[page].float() * (old / scale)[..., None, None]
    mine = torch.where(new[:, :, None, :, None], tile / scale[..., None, None], held)
    out = torch.where((new | kept)[:, :, None, :, None], encode(mine, code).float(), codes[page].float())
    codes[page] = encode(out, code)
    scales[page] = scale


def plain_attend(s):
    q, table, lens = s["q"], s["tables"], s["lens"]
    kc, ks, vc, vs = s["cache"]
    n_seqs, (n_tok, n_head, hd), n_kv = lens.numel(), q.shape, kc.shape[1]
    group = n_head // n_kv

    def values(codes, scales):
        page = table.long()
        return (codes[page].float() * scales[page][..., None, None]).transpose(1, 2).flatten(2, 3)   # [n_seqs][n_kv][cells][hd]

    cu = s["cu_q"] if s["cu_q"] is not None else torch.arange(n_seqs + 1, device=DEV, dtype=torch.int32) * s["max_q"]
    n_q = cu[1:] - cu[:-1]
    i = torch.arange(s["max_q"], device=DEV, dtype=torch.int32)
    row = (cu[:-1, None] + i).clamp(max=n_tok - 1).long()
    qp = q[row].float().view(n_seqs, s["max_q"], n_kv, group, hd).permute(0, 2, 1, 3, 4).flatten(2, 3)   # [n_seqs][n_kv][max_q * group][hd]
    see = lens[:, None] - (n_q[:, None] - 1 - i)                                                        # cells that token i sees
    k = values(kc, ks)
    dots = (qp @ k.transpose(2, 3)) * s["scale"]
    del k
    mask = torch.arange(dots.shape[3], device=DEV)[None, None, :] < see[:, :, None]
    mask = mask.repeat_interleave(group, 1)[:, None]
    dots = dots.masked_fill(~mask, float("-inf"))
    top = dots.amax(-1, keepdim=True).clamp(min=-1e30)
    e = torch.exp(dots - top)
    p = e / e.sum(-1, keepdim=True).clamp(min=1e-30)
    o = (p @ values(vc, vs)).view(n_seqs, n_kv, s["max_q"], group, hd).permute(0, 2, 1, 3, 4).reshape(n_seqs, s["max_q"], n_head, hd)
    seq = torch.searchsorted(cu, torch.arange(n_tok, device=DEV, dtype=torch.int32), right=True) - 1
    return o[seq, torch.arange(n_tok, device=DEV) - cu[seq]].to(q.dtype)


def run(s):
    op = s["op"]
    if own:
        from breccia_b200 import qsa

        if op == "rope":
            return s["rope"].apply(s["q"], s["k"], s["positions"])
        if op == "write":
            qsa.kv8_append(s["pool"], 0, s["k"], s["v"], s["tables"], s["pos0"], s["max_end"], cu_tokens=s["cu"], rope=s["rope"])
            return qsa.kv8_read(s["pool"], 0, s["tables"], s["read0"], s["max_end"], cu_tokens=s["cu_back"], total_tokens=s["total_back"],
                                dtype=s["dtype"])
        if op == "read":
            return qsa.kv8_read(s["pool"], 0, s["tables"], s["pos0"], s["max_end"], cu_tokens=s["cu"], total_tokens=s["total"], dtype=s["dtype"])
        return qsa.kv8_attend(s["pool"], 0, s["q"], s["tables"], s["lens"], s["max_end"], s["workspace"], max_q=s["max_q"], cu_q=s["cu_q"],
                              scale=s["scale"])
    if op == "rope":
        return tuple(rotate(x, s["positions"], s["rope"]).to(s["dtype"]) for x in (s["q"], s["k"]))
    if op == "attend":
        return plain_attend(s)
    kc, ks, vc, vs = s["cache"]
    if op == "write":
        k = s["k"]
        if s["rope"] is not None:
            k = rotate(k, token_cells(s["cu"], s["pos0"], s["total"])[1], s["rope"])
        plain_write(kc, ks, k, s, s["case"]["code"])
        plain_write(vc, vs, s["v"], s, s["case"]["code"])
        cu, pos0, total = s["cu_back"], s["read0"], s["total_back"]
    else:
        cu, pos0, total = s["cu"], s["pos0"], s["total"]
    return tuple(plain_read(c, x, s["tables"], cu, pos0, total, s["dtype"]) for c, x in ((kc, ks), (vc, vs)))


# ------------------------------------------------------------------------------------------------- the definition in 64 bits
def exact_rope(x, pos, n_rot, layout, scaling):
    f, m = rope_freqs(n_rot, scaling)
    z = torch.polar(torch.full_like(f, m).expand(len(pos), -1), pos.double()[:, None] * f)[:, None, :]
    out = x.double().clone()
    a = out[..., :n_rot]
    pairs = a.unflatten(-1, (2, -1)).transpose(-1, -2) if layout == "half" else a.unflatten(-1, (-1, 2))
    w = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * z)
    out[..., :n_rot] = (w.transpose(-1, -2) if layout == "half" else w).flatten(-2)
    return out


def exact_code(x, code):
    """The value of the nearest code, ties to even, in float64."""
    if code == "int8":
        return x.round().clamp(-127, 127)
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    e = torch.where(x.abs() >= torch.exp2(e + 1), e + 1, torch.where(x.abs() < torch.exp2(e), e - 1, e)).clamp(min=-6)
    step = torch.exp2(e - 3)
    return ((x / step).round() * step).clamp(-448, 448)


def exact_exponent(amax, code):
    """Least e with amax <= top * 2^e."""
    top = 448.0 if code == "e4m3" else 127.0
    e = EXP_MIN
    while e < EXP_MAX and amax > math.ldexp(top, e):
        e += 1
    return e


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    op = case["op"]
    if op == "rope":
        if case["tokens"] * (case["n_head"] + case["n_kv"]) * case["hd"] > 300_000_000:
            return None
        return tuple(exact_rope(s[n], s["positions"], case["n_rot"], case["layout"], case["scaling"]) for n in ("q", "k"))
    kc, ks, vc, vs = s["cache"]
    table = s["tables"].tolist()
    if op == "read":
        out = []
        for codes, scales in ((kc, ks), (vc, vs)):
            rows = []
            for t, n in zip(table, lengths(case)):
                at = torch.tensor(t[: pages_of(n)], device=DEV)
                rows.append((codes[at].double() * scales[at].double()[:, :, None, None]).transpose(1, 2).flatten(0, 1)[:n])
            out.append(torch.cat(rows))
        return tuple(out)
    if op == "write":
        if sum(lengths(case)) // CELLS * case["n_kv"] > 20_000:
            return None
        k, v = s["k"].double(), s["v"].double()
        out, at = ([], []), 0
        for q, (n, p) in enumerate(zip(lengths(case), starts(case))):
            rows = k[at:at + n]
            if case["rope"]:
                rows = exact_rope(rows, torch.arange(p, p + n, device=DEV), case["hd"] // 2, "half", "yarn")
            for side, (x, codes, scales) in enumerate(((rows, kc, ks), (v[at:at + n], vc, vs))):
                held = p % CELLS
                page = table[q][p // CELLS]
                old = codes[page, :, :held].double() * scales[page].double()[:, None, None]
                cells = torch.cat([old.transpose(0, 1), x])
                parts = []
                for i in range(0, held + n, CELLS):
                    part = cells[i:i + CELLS].clone()
                    fresh = part[held:] if i == 0 else part
                    amax = fresh.abs().amax((0, 2)).tolist()
                    e = [exact_exponent(a, case["code"]) for a in amax]
                    if i == 0 and held:
                        e = [max(a, int(b)) for a, b in zip(e, torch.log2(scales[page].double()).round().tolist())]
                    unit = torch.exp2(torch.tensor(e, dtype=torch.float64, device=DEV))[None, :, None]
                    parts.append(exact_code(part / unit, case["code"]) * unit)
                out[side].append(torch.cat(parts))
            at += n
        return tuple(torch.cat(o) for o in out)
    if sum(lengths(case)) * case["n_kv"] * case["hd"] > 1_500_000_000:
        return None
    rows, at, group = [], 0, case["n_head"] // case["n_kv"]
    for t, n, nq in zip(table, lengths(case), q_lengths(case)):
        ids = torch.tensor(t[: pages_of(n)], device=DEV)
        k, v = ((c[ids].double() * x[ids].double()[:, :, None, None]).transpose(1, 2).flatten(0, 1)[:n] for c, x in ((kc, ks), (vc, vs)))
        for i in range(nq):
            see = n - (nq - 1 - i)
            q = s["q"][at].double().unflatten(0, (-1, group))
            at += 1
            if see <= 0:
                rows.append(torch.zeros(case["n_head"], case["hd"], dtype=torch.float64, device=DEV))
                continue
            d = torch.einsum("hgd,chd->hgc", q, k[:see]) * s["scale"]
            rows.append(torch.einsum("hgc,chd->hgd", torch.softmax(d, -1), v[:see]).flatten(0, 1))
    return torch.stack(rows)
