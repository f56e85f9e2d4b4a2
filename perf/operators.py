"""Rotary positions and the 4-bit key/value cache as timed cases.

Five paths, each in its plain form (elementary torch operations) and, where
``own`` is true, through the entry points a program calls:

* ``rope``   -- rotary positions on the heads of some tokens (``DeviceOps.rope``);
* ``append`` -- new keys (rotated on the way) and values written into the paged
  4-bit cache and read back (``kv4_append``, ``kv4_read``);
* ``attn``   -- attention over the cache, the new rows at its end
  (``kv4_attention``): one token, decode lanes, prompts;
* ``weigh``  -- the attention weight that each cached slot received, added to
  its running sum (``kv4_weigh``);
* ``evict``  -- the heaviest slots kept, in order, in new pages
  (``kv4_evict``), with the kept cache read back.

The cache: pages of 64 slots; in a page, per kv head, 80 * D bytes: key codes
(32 D), value codes (32 D), key scales (8 D), value scales (8 D).  Every 32
values of a token's head share a scale d (f16 of 7 significant bits) and a
minimum m (f16); a 4-bit code q stands for d q + m.

  * eight codes make a dword, code j at bit (6, 22, 2, 18, 14, 30, 10, 26)[j]
    of it, modulo 32;
  * key codes: [tile of 16 tokens][group quad][lane = 16 kg + token][group in
    quad], the dword's codes being dims 32 group + 8 kg + 0..7 (a head of 64
    has one "quad" of two groups);
  * value codes: [block of 32 tokens][64 dims][lane = 16 rg + dim % 16][dim /
    16 % 4], the dword's codes being tokens 4 rg + 0..3 and 16 + 4 rg + 0..3;
  * key scales: [token][d of each group, then m of each group];
  * value scales: [block of 32 tokens][d, then m][group][token in the order of
    the value codes: rg, half of the block, 0..3].
"""
import math

import torch

own = False

PAGE = 64
BITS = (6, 22, 2, 18, 14, 30, 10, 26)
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TYPE_CODE = {"f32": 0, "f16": 1, "bf16": 2}

# Rotations by name: rot_dim is a case's own.  "plain" is the 8B decoder's,
# "long" its long-context form with frequency bands, "yarn" a blend of two.
SCALINGS = {
    "plain": {"base": 500000.0, "scaling": "none"},
    "linear": {"base": 10000.0, "scaling": "linear", "factor": 4.0},
    "long": {"base": 500000.0, "scaling": "bands", "factor": 8.0, "low": 1.0, "high": 4.0, "context": 8192},
    "yarn": {"base": 1000000.0, "scaling": "yarn", "factor": 4.0, "low": 1.0, "high": 32.0, "context": 32768},
}


def listed():
    return [
        # The q and k heads (32 + 8) of one token of an 8B decoder.
        {"name": "rope_t1", "path": "rope", "type": "f32", "tokens": 1, "heads": 40, "dim": 128, "rot": 128,
         "layout": "half", "scaling": "plain", "start": 1000},
        # A prompt of odd length in bf16, half of each head rotated, far positions.
        {"name": "rope_prompt_4001", "path": "rope", "type": "bf16", "tokens": 4001, "heads": 72, "dim": 128,
         "rot": 64, "layout": "interleaved", "scaling": "yarn", "start": 120000},
        # 32 decode lanes write their token.
        {"name": "append_b32", "path": "append", "type": "f32", "seqs": 32, "rows_lo": 1, "rows": 1, "len": 8000,
         "kv": 8, "dim": 128, "layout": "half", "scaling": "plain"},
        # Three prompts of different lengths, one of which continues a cache.
        {"name": "append_prompts", "path": "append", "type": "bf16", "seqs": 3, "rows_lo": 801, "rows": 4100,
         "len": 4500, "kv": 8, "dim": 128, "layout": "half", "scaling": "long"},
        # One token of the 8B decoder, early in a conversation.
        {"name": "attn_t1_777", "path": "attn", "type": "f32", "seqs": 1, "rows_lo": 1, "rows": 1, "len_lo": 777,
         "len": 777, "heads": 32, "kv": 8, "dim": 128, "window": 0},
        # One token at the end of a long document.
        {"name": "attn_t1_130001", "path": "attn", "type": "f32", "seqs": 1, "rows_lo": 1, "rows": 1,
         "len_lo": 130001, "len": 130001, "heads": 32, "kv": 8, "dim": 128, "window": 0},
        # 64 decode lanes of a 70B decoder (8 queries to a kv head), lengths 1 to 8000.
        {"name": "attn_b64", "path": "attn", "type": "bf16", "seqs": 64, "rows_lo": 1, "rows": 1, "len_lo": 1,
         "len": 8000, "heads": 64, "kv": 8, "dim": 128, "window": 0},
        # A chunk of a prompt behind what is already cached.
        {"name": "attn_chunk_2000", "path": "attn", "type": "f32", "seqs": 1, "rows_lo": 2000, "rows": 2000,
         "len_lo": 6000, "len": 6000, "heads": 32, "kv": 8, "dim": 128, "window": 0},
        # Three whole prompts of different lengths.
        {"name": "attn_prompts_bf16", "path": "attn", "type": "bf16", "seqs": 3, "rows_lo": 900, "rows": 4097,
         "len_lo": 900, "len": 4097, "heads": 64, "kv": 8, "dim": 128, "window": 0},
        # 32 decode lanes add the weights of their token.
        {"name": "weigh_b32", "path": "weigh", "type": "f32", "seqs": 32, "rows_lo": 1, "rows": 1, "len_lo": 2000,
         "len": 8000, "heads": 32, "kv": 8, "dim": 128, "window": 0},
        # The weights that the last 64 rows of a prompt give, in bf16.
        {"name": "weigh_rows_64", "path": "weigh", "type": "bf16", "seqs": 1, "rows_lo": 64, "rows": 64,
         "len_lo": 32000, "len": 32000, "heads": 64, "kv": 8, "dim": 128, "window": 0},
        # 16 lanes shrink to a quarter of their cache.
        {"name": "evict_b16", "path": "evict", "type": "bf16", "seqs": 16, "len_lo": 1500, "len": 8000, "kv": 8,
         "dim": 128, "keep": 2000, "first": 4, "recent": 256},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    path = rng.choice(["rope", "append", "attn", "attn", "attn", "weigh", "evict"])
    ty = rng.choice(["f32", "f32", "bf16", "f16"])
    dim = rng.choice([64, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 8])
    scaling = rng.choice(sorted(SCALINGS))
    layout = rng.choice(["half", "interleaved"])
    if path == "rope":
        heads = rng.randint(1, 72)
        return {"path": "rope", "type": ty, "tokens": max(1, min(_log_int(rng, 1, 16384), 36000000 // (heads * dim))),
                "heads": heads, "dim": dim, "rot": rng.choice([dim, dim, dim // 2, 32]), "layout": layout,
                "scaling": scaling, "start": _log_int(rng, 1, 500000)}
    if path == "append":
        seqs = _log_int(rng, 1, 64)
        top = max(1, 7000 * 8 * 128 // (seqs * kv * dim))
        rows = _log_int(rng, 1, min(top, 8000))
        return {"path": "append", "type": ty, "seqs": seqs, "rows_lo": rng.randint(1, rows), "rows": rows,
                "len": rows + rng.randint(0, 4000), "kv": kv, "dim": dim, "layout": layout, "scaling": scaling}
    if path == "evict":
        seqs = _log_int(rng, 1, 16)
        top = 16 * 8000 * 8 * 128 // (seqs * kv * dim)
        n = _log_int(rng, 300, min(top, 32000))
        keep = rng.randint(64, max(65, n // 2))
        first = rng.randint(0, 8)
        return {"path": "evict", "type": ty, "seqs": seqs, "len_lo": rng.randint(1, n), "len": n, "kv": kv,
                "dim": dim, "keep": keep, "first": first, "recent": rng.randint(0, keep - first)}
    group = rng.choice([1, 2, 4, 4, 8])
    c = {"path": path, "type": ty, "seqs": 1, "rows_lo": 1, "rows": 1, "len_lo": 1, "len": 1, "heads": kv * group,
         "kv": kv, "dim": dim, "window": rng.choice([0, 0, 0, 1000])}
    if path == "weigh" or rng.random() < 0.6:  # decode lanes, or the last rows of a prompt
        c["seqs"] = _log_int(rng, 1, 64)
        c["rows"] = rng.choice([1, 1, 2, 7]) if path == "attn" else rng.choice([1, 1, 5, 32])
        top = 64 * 8000 * 8 * 128 // (c["seqs"] * kv * dim * 2)
        c["len"] = c["rows"] + _log_int(rng, 1, min(top, 130000))
    else:
        c["seqs"] = rng.randint(1, 4)
        c["rows"] = _log_int(rng, 20, 4000 // c["seqs"])
        c["len"] = c["rows"] + rng.randint(0, 2000)
    c["rows_lo"] = rng.randint(1, c["rows"])
    c["len_lo"] = rng.randint(1, c["len"])
    return c


# ---- sizes that follow from a case -----------------------------------------

def _spread(lo, hi, n):
    """n whole numbers from hi down to lo."""
    return [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _rows(c):
    return _spread(c["rows_lo"], c["rows"], c["seqs"])


def _lens(c):
    """Cache lengths after the new rows; a length never falls below its rows."""
    if c["path"] == "append":
        spare = c["len"] - c["rows"]
        return [r + (spare if i % 3 == 1 or c["rows"] == 1 else 0) for i, r in enumerate(_rows(c))]
    lens = _spread(c["len_lo"], c["len"], c["seqs"])
    return lens if c["path"] == "evict" else [max(n, r) for n, r in zip(lens, _rows(c))]


def _seen(n, rows, window):
    """Keys that the last `rows` of n tokens see, all together."""
    if not window:
        return rows * n - rows * (rows - 1) // 2
    return sum(min(p + 1, window) for p in range(n - rows, n))


def _pages(n):
    return -(-n // PAGE)


def inv_freq(rot, base, scaling, factor=1.0, low=0.0, high=0.0, context=0):
    """(angle per position of each pair, magnitude) of a rotation."""
    f = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
    if scaling == "linear":
        return [v / factor for v in f], 1.0
    if scaling == "bands":
        out = []
        for v in f:
            turns = context * v / (2 * math.pi)  # over the trained context
            s = min(1.0, max(0.0, (turns - low) / (high - low)))
            out.append((1 - s) * v / factor + s * v)
        return out, 1.0
    if scaling == "yarn":
        def at(turns):
            return rot * math.log(context / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(math.floor(at(high)), 0), min(math.ceil(at(low)), rot - 1)
        out = []
        for i, v in enumerate(f):
            ramp = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            out.append(v / factor * ramp + v * (1 - ramp))
        return out, 0.1 * math.log(factor) + 1.0
    return f, 1.0


# ---- inputs ----------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", dtype=torch.float32, generator=g)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _starts(rows):
    return _ints([sum(rows[:i]) for i in range(len(rows) + 1)])


def _random_pages(g, n, kv, dim):
    """n pages of keys and values that are roughly N(0, 1): uint8 [n][kv][80 dim]."""
    page = torch.empty(n, kv, 80 * dim, dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 25) // (kv * 64 * dim))
    for i in range(0, n, step):
        m = min(step, n - i)
        q = (_randn(g, m, kv, 64 * dim, 2) * 2.8 + 7.5).round_().clamp_(0, 15).to(torch.uint8)
        page[i:i + m, :, :64 * dim] = q[..., 0] | (q[..., 1] << 4)
    # Scales of 7 significant bits around 1/2.8, minima around -7.5 of them.
    # In key scales the minima of a token follow its scales, in value scales
    # the minima of a block follow its scales.
    groups = dim // 32
    for at, runs, width in ((64 * dim, 64, groups), (72 * dim, 2, 32 * groups)):
        d = (64 + torch.randint(0, 64, (n, kv, runs, width), device="cuda", generator=g)).float() / 256
        mn = -7.5 * d + 0.2 * _randn(g, n, kv, runs, width)
        both = torch.stack([d, mn], 3).to(torch.float16)
        page[:, :, at:at + 8 * dim] = both.reshape(n, kv, -1).view(torch.uint8)
    return page


def _table(g, seqs, width, pool):
    """A page table whose pages lie anywhere in the pool."""
    return torch.randperm(pool, device="cuda", generator=g)[:seqs * width].view(seqs, width).to(torch.int32).contiguous()


def prepare(case, seed):
    c, g = case, _generator(seed)
    ty = TYPES[c["type"]]
    st = {"case": c}
    if c["path"] == "rope":
        shape = (c["tokens"], c["heads"], c["dim"])
        st.update(x=_randn(g, *shape).to(ty), y=torch.empty(shape, dtype=ty, device="cuda"),
                  pos=c["start"] + torch.arange(c["tokens"], dtype=torch.int32, device="cuda"))
        return st
    lens, kv, dim = _lens(c), c["kv"], c["dim"]
    width = max(_pages(n) for n in lens)
    pool = c["seqs"] * width + 7
    st.update(len=_ints(lens), table=_table(g, c["seqs"], width, pool))
    if c["path"] == "append":
        rows = _rows(c)
        n = sum(rows)
        pos = [torch.arange(m - r, m, dtype=torch.int32, device="cuda") for m, r in zip(lens, rows)]
        # Some key channels are far from the others, as in trained models.
        k = _randn(g, n, kv, dim) * torch.exp(0.7 * _randn(g, kv, dim)) + _randn(g, kv, dim)
        st.update(start=_starts(rows), pos=torch.cat(pos), k=k.to(ty), v=_randn(g, n, kv, dim).to(ty),
                  pages=torch.zeros(pool, kv, 80 * dim, dtype=torch.uint8, device="cuda"),
                  k_out=torch.empty(n, kv, dim, dtype=ty, device="cuda"),
                  v_out=torch.empty(n, kv, dim, dtype=ty, device="cuda"))
        return st
    st["pages"] = _random_pages(g, pool, kv, dim)
    if c["path"] == "evict":
        # Attention weight is heavy-tailed; sums of few terms coincide.
        acc = torch.exp(2.0 * _randn(g, c["seqs"], kv, width * PAGE))
        st["acc"] = torch.where(acc < 0.5, (acc * 16).round() / 16, acc)
        keep = c["keep"]
        rows = [min(n, keep) for n in lens]
        wide = _pages(max(rows))
        st.update(kept_start=_starts(rows), kept=sum(rows), kept_table=_table(g, c["seqs"], wide, c["seqs"] * wide),
                  kept_pages=torch.zeros(c["seqs"] * wide, kv, 80 * dim, dtype=torch.uint8, device="cuda"),
                  new_len=torch.empty(c["seqs"], dtype=torch.int32, device="cuda"),
                  idx=torch.empty(c["seqs"], kv, keep, dtype=torch.int32, device="cuda"),
                  acc_out=torch.empty(c["seqs"], kv, keep, device="cuda"),
                  k_out=torch.empty(sum(rows), kv, dim, dtype=ty, device="cuda"),
                  v_out=torch.empty(sum(rows), kv, dim, dtype=ty, device="cuda"))
        return st
    rows = _rows(c)
    n = sum(rows)
    # Queries long enough for scores of standard deviation 2.
    st.update(start=_starts(rows), rows=rows, n=n, max_rows=max(rows), q=(2.0 * _randn(g, n, c["heads"], dim)).to(ty))
    if c["path"] == "attn":
        st.update(out=torch.empty(n, c["heads"], dim, dtype=ty, device="cuda"),
                  lse=torch.empty(n, c["heads"], device="cuda"))
    else:
        st.update(acc=torch.rand(c["seqs"], kv, width * PAGE, device="cuda", generator=g),
                  acc_out=torch.zeros(c["seqs"], kv, width * PAGE, device="cuda"))
        # What the attention call of the same rows has returned: about the log
        # of the keys seen, with the spread of the scores.
        seen = torch.cat([torch.arange(m - r, m, device="cuda") for m, r in zip(lens, rows)]).float() + 1
        st["lse"] = (torch.log(seen)[:, None] + 2.0 + 0.3 * _randn(g, n, c["heads"])).contiguous()
    return st


# ---- the plain forms -------------------------------------------------------

def _codes(words):
    """int32 dwords [...] -> their eight codes [..., 8], f32."""
    w = words.unsqueeze(-1)
    at = torch.tensor(BITS, dtype=torch.int32, device=w.device)
    low = (w >> at) & 15
    wrapped = ((w >> 30) & 3) | ((w & 3) << 2)
    return torch.where(at == 30, wrapped, low).to(torch.float32)


def _plain_keys(page, dim):
    """f32 [n][kv][64][dim] of pages [n][kv][80 dim]."""
    n, kv, groups = page.shape[0], page.shape[1], dim // 32
    quad = min(groups, 4)
    w = page[:, :, :32 * dim].contiguous().view(torch.int32).view(n, kv, 4, groups // quad, 4, 16, quad)
    q = _codes(w).permute(0, 1, 2, 5, 3, 6, 4, 7).reshape(n, kv, 64, groups, 32)
    s = page[:, :, 64 * dim:72 * dim].contiguous().view(torch.float16).view(n, kv, 64, 2, groups, 1).float()
    return (q * s[:, :, :, 0] + s[:, :, :, 1]).reshape(n, kv, 64, dim)


def _plain_values(page, dim):
    n, kv, groups = page.shape[0], page.shape[1], dim // 32
    w = page[:, :, 32 * dim:64 * dim].contiguous().view(torch.int32).view(n, kv, 2, dim // 64, 4, 16, 4)
    q = _codes(w).view(n, kv, 2, dim // 64, 4, 16, 4, 2, 4).permute(0, 1, 2, 7, 4, 8, 3, 6, 5)
    s = page[:, :, 72 * dim:].contiguous().view(torch.float16).view(n, kv, 2, 2, groups, 4, 2, 4).float()
    s = s.permute(0, 1, 3, 2, 6, 5, 7, 4).reshape(n, kv, 2, 64, groups, 1)
    q = q.reshape(n, kv, 64, groups, 32)
    return (q * s[:, :, 0] + s[:, :, 1]).reshape(n, kv, 64, dim)


def _gathered(st, what):
    """f32 [seqs][kv][slots][dim] of a cache's keys or values."""
    c = st["case"]
    seqs, width = st["table"].shape
    v = what(st["pages"][st["table"].long().reshape(-1)], c["dim"])
    return v.view(seqs, width, c["kv"], PAGE, c["dim"]).permute(0, 2, 1, 3, 4).reshape(seqs, c["kv"], width * PAGE,
                                                                                    c["dim"])


def _plain_rope(x, pos, rot, layout, scaling, wide):
    """Rotated f32 x [rows][heads][dim]; angles in 64 bits, and (wide) the
    products too."""
    f, mag = inv_freq(rot, **SCALINGS[scaling])
    a = pos.double()[:, None, None] * torch.tensor(f, dtype=torch.float64, device=x.device)
    cos, sin = torch.cos(a) * mag, torch.sin(a) * mag
    x = x.double() if wide else x.float()
    cos, sin = cos.to(x.dtype), sin.to(x.dtype)
    r = x[..., :rot]
    u, w = (r[..., :rot // 2], r[..., rot // 2:]) if layout == "half" else (r[..., 0::2], r[..., 1::2])
    p, q = u * cos - w * sin, u * sin + w * cos
    r = torch.cat([p, q], -1) if layout == "half" else torch.stack([p, q], -1).flatten(-2)
    return torch.cat([r, x[..., rot:]], -1).float()


def _plain_quantised(x):
    """The values that 4-bit codes of x [...][dim] stand for, f32."""
    g = x.unflatten(-1, (-1, 32)).double()
    m = g.amin(-1, keepdim=True).float().to(torch.float16).double()
    r = (g.amax(-1, keepdim=True) - m) / 15.0
    step = torch.exp2(torch.clamp(torch.frexp(r.clamp(min=2.0 ** -30))[1] - 7, min=-24).double())
    d = torch.where(r > 0, torch.ceil(r / step) * step, torch.zeros_like(r))
    q = torch.where(d > 0, torch.round((g - m) / torch.where(d > 0, d, torch.ones_like(d))), torch.zeros_like(g))
    return (d * q.clamp(0, 15) + m).float().flatten(-2)


def _row_of(st, tensor):
    """[n][...] rows -> [seqs][max_rows][...], and where a row is one."""
    rows = st["start"][1:] - st["start"][:-1]
    i = torch.arange(st["max_rows"], device="cuda")
    at = (st["start"][:-1, None] + i).clamp(max=st["n"] - 1).long()
    return tensor[at], i < rows[:, None], rows


def _plain_scores(st):
    """Masked scores [seqs][kv][group x max_rows][slots], f32, in natural units."""
    c = st["case"]
    seqs, kv, dim = c["seqs"], c["kv"], c["dim"]
    q, real, rows = _row_of(st, st["q"].float())
    group = c["heads"] // kv
    q = q.view(seqs, -1, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kv, -1, dim)
    s = torch.matmul(q / math.sqrt(dim), _gathered(st, _plain_keys).transpose(2, 3).contiguous())
    slot = torch.arange(s.shape[-1], device="cuda")
    pos = (st["len"] - rows)[:, None] + torch.arange(st["max_rows"], device="cuda")
    hide = (slot > pos[..., None]) | ~real[..., None]
    if c["window"]:
        hide |= slot <= pos[..., None] - c["window"]
    s = s.view(seqs, kv, group, st["max_rows"], -1)
    return s.masked_fill_(hide[:, None, None], -math.inf), real


def _flat_rows(x, real):
    """[seqs][kv][group][rows][...] -> [n][heads][...] of the real rows."""
    x = x.movedim(3, 1).flatten(2, 3)
    return x[real]


def _plain_run(st):
    c = st["case"]
    ty = TYPES[c["type"]]
    if c["path"] == "rope":
        return _plain_rope(st["x"], st["pos"], c["rot"], c["layout"], c["scaling"], False).to(ty)
    if c["path"] == "append":
        k = _plain_rope(st["k"], st["pos"], c["dim"], c["layout"], c["scaling"], True)
        return [_plain_quantised(k).to(ty), _plain_quantised(st["v"].float()).to(ty)]
    if c["path"] == "evict":
        return _plain_evict(st)
    s, real = _plain_scores(st)
    if c["path"] == "weigh":
        lse, _, _ = _row_of(st, st["lse"])
        lse = lse.view(c["seqs"], -1, c["kv"], c["heads"] // c["kv"]).permute(0, 2, 3, 1)
        return st["acc"] + torch.exp(s - lse[..., None]).sum((2, 3))
    top = s.amax(-1, keepdim=True).clamp(min=-1e30)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), _gathered(st, _plain_values)).view(*p.shape[:4], c["dim"])
    o = o / torch.where(total > 0, total, torch.ones_like(total))
    return [_flat_rows(o, real).to(ty), _flat_rows(torch.log(total) + top, real)[..., 0]]


def _plain_evict(st):
    c = st["case"]
    keep, slots = c["keep"], st["acc"].shape[2]
    at = torch.arange(slots, device="cuda")
    n = st["len"].long()[:, None]
    always = (at < c["first"]) | (at >= n - c["recent"]) | (n <= keep)
    key = torch.where(always[:, None], math.inf, st["acc"].clamp(min=0)).masked_fill((at >= n)[:, None], -1.0)
    order = torch.sort(key, dim=-1, descending=True, stable=True)[1][..., :keep]
    fits = torch.arange(keep, device="cuda") < n
    idx = torch.sort(torch.where(fits[:, None], order, slots), -1)[0]
    there = idx < slots
    safe = idx.clamp(max=slots - 1)
    acc = torch.where(there, torch.gather(st["acc"], 2, safe), torch.zeros((), device="cuda"))
    out = [torch.where(there, idx, -1).to(torch.int32), acc]
    for what in (_plain_keys, _plain_values):
        v = torch.gather(_gathered(st, what), 2, safe[..., None].expand(-1, -1, -1, c["dim"]))
        out.append(v.permute(0, 2, 1, 3)[fits].to(TYPES[c["type"]]))
    return out


# ---- the framework's calls -------------------------------------------------

def _kept(st, name, make):
    """What a program makes once and keeps: handles and workspaces."""
    if name not in st:
        st[name] = make()
    return st[name]


def _rope_handle(aa, c, rot):
    return aa.Rope(rot, layout=c["layout"], **SCALINGS[c["scaling"]])


def _cache(aa, c, pages, table):
    return aa.KV4Cache(c["dim"], c["kv"], pages.shape[0], table.shape[1], pages.data_ptr(), table.data_ptr())


def _own_run(st):
    import aspida_amd as aa
    c = st["case"]
    sp = torch.cuda.current_stream().cuda_stream
    dev = _kept(st, "dev", aa.DeviceOps)
    ty, dim = TYPE_CODE[c["type"]], c["dim"]
    if c["path"] == "rope":
        rope = _kept(st, "rope", lambda: _rope_handle(aa, c, c["rot"]))
        row = c["heads"] * dim
        dev.rope(rope, ty, st["x"].data_ptr(), row, c["tokens"], c["heads"], dim, st["pos"].data_ptr(),
                 st["y"].data_ptr(), row, sp)
        return st["y"]
    cache = _kept(st, "cache", lambda: _cache(aa, c, st["pages"], st["table"]))
    kv, seqs = c["kv"], c["seqs"]
    if c["path"] == "append":
        rope = _kept(st, "rope", lambda: _rope_handle(aa, c, dim))
        n, row = st["k"].shape[0], kv * dim
        dev.kv4_append(cache, ty, st["k"].data_ptr(), row, st["v"].data_ptr(), row, n, seqs, st["start"].data_ptr(),
                       st["len"].data_ptr(), rope, st["pos"].data_ptr(), sp)
        dev.kv4_read(cache, ty, n, seqs, st["start"].data_ptr(), st["len"].data_ptr(), st["k_out"].data_ptr(), row,
                     st["v_out"].data_ptr(), row, sp)
        return [st["k_out"], st["v_out"]]
    if c["path"] == "evict":
        kept = _kept(st, "kept_cache", lambda: _cache(aa, c, st["kept_pages"], st["kept_table"]))
        row = kv * dim
        dev.kv4_evict(cache, seqs, st["len"].data_ptr(), st["acc"].data_ptr(), st["acc"].shape[2], c["keep"],
                      c["first"], c["recent"], kept, st["new_len"].data_ptr(), st["idx"].data_ptr(),
                      st["acc_out"].data_ptr(), sp)
        dev.kv4_read(kept, ty, st["kept"], seqs, st["kept_start"].data_ptr(), st["new_len"].data_ptr(),
                     st["k_out"].data_ptr(), row, st["v_out"].data_ptr(), row, sp)
        return [st["idx"], st["acc_out"], st["k_out"], st["v_out"]]
    heads, row = c["heads"], c["heads"] * dim
    scale = 1.0 / math.sqrt(dim)
    if c["path"] == "weigh":
        dev.kv4_weigh(cache, ty, st["q"].data_ptr(), row, heads, st["n"], seqs, st["start"].data_ptr(),
                      st["max_rows"], st["len"].data_ptr(), scale, st["lse"].data_ptr(), st["acc"].data_ptr(),
                      st["acc_out"].data_ptr(), st["acc"].shape[2], sp, window=c["window"])
        return st["acc_out"]
    work = _kept(st, "work", lambda: torch.empty(
        dev.kv4_attention_work_bytes(cache, heads, st["n"], seqs, st["max_rows"]), dtype=torch.uint8, device="cuda"))
    dev.kv4_attention(cache, ty, st["q"].data_ptr(), row, heads, st["n"], seqs, st["start"].data_ptr(),
                      st["max_rows"], st["len"].data_ptr(), scale, st["out"].data_ptr(), row, work.data_ptr(), sp,
                      window=c["window"], lse=st["lse"].data_ptr())
    return [st["out"], st["lse"]]


def run(st):
    return _own_run(st) if own else _plain_run(st)


# ---- what a pass cannot do without -----------------------------------------

def work(case):
    c = case
    size, dim = 4 if c["type"] == "f32" else 2, c["dim"]
    if c["path"] == "rope":
        n = c["tokens"] * c["heads"]
        return {"bytes": 2 * size * n * dim + 4 * c["tokens"], "flops": 3 * n * c["rot"]}
    kv, lens = c["kv"], _lens(c)
    token = kv * dim  # a token's keys, or its values; 5 bits each in the cache
    if c["path"] == "append":
        n = sum(_rows(c))
        return {"bytes": n * token * (4 * size + 2 * 5 / 8) + 4 * n, "flops": n * token * 9}
    if c["path"] == "evict":
        kept = sum(min(n, c["keep"]) for n in lens)
        return {"bytes": 4 * kv * sum(lens) + 8 * kv * c["seqs"] * c["keep"] + kept * token * (4 * 5 / 8 + 2 * size),
                "flops": kept * token * 4}
    rows = _rows(c)
    seen = sum(_seen(n, r, c["window"]) for n, r in zip(lens, rows))
    there = sum(min(n, c["window"] + r - 1) if c["window"] else n for n, r in zip(lens, rows))
    q = sum(rows) * c["heads"] * (dim * size + 4)
    if c["path"] == "weigh":
        return {"bytes": int(there * token * 5 / 8 + q + 8 * kv * there), "flops": 2 * dim * c["heads"] * seen}
    return {"bytes": int(2 * there * token * 5 / 8 + 2 * q), "flops": 4 * dim * c["heads"] * seen}


# ---- the same in 64 bits ---------------------------------------------------

def _exact_cache(st, b, kind):
    """f64 [kv][slots][dim] of sequence b, token by token and dim by dim from the layout's addresses."""
    c = st["case"]
    dim, dev = c["dim"], "cuda"
    page = st["pages"][st["table"][b].long()]
    tok, col = torch.arange(PAGE, device=dev)[:, None], torch.arange(dim, device=dev)[None, :]
    groups = dim // 32
    grp, kg, j = col // 32, col % 32 // 8, col % 8
    half = page.contiguous().view(torch.float16)
    if kind == "k":
        quad = min(groups, 4)
        word = tok // 16 * (2 * dim) + grp // quad * (64 * quad) + (16 * kg + tok % 16) * quad + grp % quad
        sd = 32 * dim + tok * 2 * groups + grp
        sm = sd + groups
        pos = j
    else:
        rg, hi, lo = tok % 16 // 4, tok % 32 // 16, tok % 4
        word = 8 * dim + tok // 32 * (4 * dim) + col // 64 * 256 + (16 * rg + col % 16) * 4 + col // 16 % 4
        sd = 36 * dim + tok // 32 * (64 * groups) + grp * 32 + rg * 8 + hi * 4 + lo
        sm = sd + 32 * groups
        pos = (4 * hi + lo).expand(PAGE, dim)
    bit = torch.tensor(BITS, device=dev)[pos].expand(PAGE, dim)
    byte = page.long()
    flat = lambda t: t.expand(PAGE, dim).reshape(-1)  # noqa: E731
    q = torch.zeros(page.shape[0], page.shape[1], PAGE * dim, dtype=torch.int64, device=dev)
    for k in range(4):  # one bit after the other
        at = (bit + k) % 32
        q += ((byte[:, :, flat(4 * word + at // 8)] >> flat(at % 8)) & 1) << k
    v = q.double() * half[:, :, flat(sd)].double() + half[:, :, flat(sm)].double()
    return v.view(-1, c["kv"], PAGE, dim).transpose(0, 1).reshape(c["kv"], -1, dim)


def _exact_rotated(x, pos, rot, layout, scaling):
    f, mag = inv_freq(rot, **SCALINGS[scaling])
    a = torch.outer(pos.double(), torch.tensor(f, dtype=torch.float64, device="cuda"))
    i = torch.arange(rot // 2, device="cuda")
    first, second = (i, i + rot // 2) if layout == "half" else (2 * i, 2 * i + 1)
    y = x.double().clone()
    turn = torch.polar(torch.full_like(a, mag), a)[:, None] * torch.complex(x[..., first].double(), x[..., second].double())
    y[..., first], y[..., second] = turn.real, turn.imag
    return y


def _exact_quantised(x):
    """f64 values of the 4-bit codes of f32 x [n][kv][dim]."""
    g = x.double().reshape(-1, 32)
    m = g.min(1).values.float().half().double()
    r = (g.max(1).values - m) / 15
    # Candidates of every exponent: the smallest multiple of 2^e that holds r
    # with at most 7 bits, from the finest step up.
    d = torch.full_like(r, math.inf)
    for e in range(8, -25, -1):
        up = torch.ceil(r * 2.0 ** -e)
        d = torch.where(up < 128, up * 2.0 ** e, d)
    d = torch.where(r > 0, d, 0.0)
    q = torch.where(d[:, None] > 0, torch.round((g - m[:, None]) / d[:, None]), 0.0).clamp(0, 15)
    return (q * d[:, None] + m[:, None]).view(x.shape)


def exact(case, seed):
    st = prepare(case, seed)
    c = case
    if c["path"] == "rope":
        return _exact_rotated(st["x"], st["pos"], c["rot"], c["layout"], c["scaling"])
    if c["path"] == "append":
        k = _exact_rotated(st["k"], st["pos"], c["dim"], c["layout"], c["scaling"]).float()
        return [_exact_quantised(k), _exact_quantised(st["v"].float())]
    lens, kv, dim = _lens(c), c["kv"], c["dim"]
    if c["path"] == "evict":
        accs, ks, vs = [], [], []
        for b, n in enumerate(lens):
            a = st["acc"][b, :, :n].double()
            if n > c["keep"]:
                rank = a.clone()
                rank[:, :c["first"]] = math.inf
                rank[:, n - c["recent"]:] = math.inf
                order = torch.argsort(-rank, dim=1, stable=True)
                idx = order[:, :c["keep"]].sort(1).values
            else:
                idx = torch.arange(n, device="cuda").expand(kv, n)
            row = torch.zeros(kv, c["keep"], dtype=torch.float64, device="cuda")
            row[:, :idx.shape[1]] = a.gather(1, idx)
            accs.append(row)
            for kind, to in (("k", ks), ("v", vs)):
                x = _exact_cache(st, b, kind)
                to.append(x.gather(1, idx[..., None].expand(-1, -1, dim)).transpose(0, 1))
        return [None, torch.stack(accs), torch.cat(ks), torch.cat(vs)]
    outs, lses, acc, at = [], [], st["acc"].double() if c["path"] == "weigh" else None, 0
    for b, (n, r) in enumerate(zip(lens, st["rows"])):
        k = _exact_cache(st, b, "k")[:, :n]
        v = _exact_cache(st, b, "v")[:, :n] if c["path"] == "attn" else None
        for lo in range(0, r, 256):
            hi = min(r, lo + 256)
            q = st["q"][at + lo:at + hi].double().view(hi - lo, kv, -1, dim)
            slot = torch.arange(n, device="cuda")
            pos = torch.arange(n - r + lo, n - r + hi, device="cuda")[:, None]
            see = slot <= pos
            if c["window"]:
                see &= slot > pos - c["window"]
            o, ls = [], []
            for h in range(kv):
                s = (q[:, h].reshape(-1, dim) @ k[h].t().contiguous() / math.sqrt(dim)).view(hi - lo, -1, n)
                s = s.masked_fill(~see[:, None], -math.inf)
                if c["path"] == "weigh":
                    lse = st["lse"][at + lo:at + hi].double().view(hi - lo, kv, -1)[:, h]
                    acc[b, h, :n] += torch.exp(s - lse[..., None]).sum((0, 1))
                else:
                    ls.append(torch.logsumexp(s, 2))
                    o.append((torch.exp(s - ls[-1][..., None]).view(-1, n) @ v[h]).view(hi - lo, -1, dim))
            if c["path"] == "attn":
                outs.append(torch.stack(o, 1).flatten(1, 2))
                lses.append(torch.stack(ls, 1).flatten(1, 2))
        at += r
    return acc if c["path"] == "weigh" else [torch.cat(outs), torch.cat(lses)]
